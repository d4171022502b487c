// linear8.h -- what the products of 8-bit matrices are called with (not part of
// the public ABI).
#pragma once

#include "rows8.h"

namespace ember {

struct Linear8Args {
    Rows8 a, w;  // n x k and m x k; a gated layer's w is 2m x k, the gate's rows first
    const float *bias, *residual;
    float *out;  // n x m
    int n, m, act;
};

}  // namespace ember
