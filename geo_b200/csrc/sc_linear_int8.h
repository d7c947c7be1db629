// 8-bit matrix product: what its two kernels share (sc_linear_int8.cu, sc_linear_int8_tc.cu).
#pragma once

#include "sc_rows8.h"

namespace geo {

struct LinearParams {
    const int8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    void *out;
    long long x_stride, w_stride, out_stride;
    int m, n, k;
};

// The tcgen05 kernel; any m, n and k (rows on 16-byte boundaries).
int launch_linear_int8_tc(const LinearParams &p, int dtype, cudaStream_t s);
// Bounded barrier waits of it that ran out since the library was loaded.
int linear_int8_tc_error_count(int *count);

}  // namespace geo
