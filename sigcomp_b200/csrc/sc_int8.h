// The int8 operators with a scale for each token and channel (sc_int8.cu), as sc_capi.cu calls them.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/sigcomp_b200.h"

namespace sc {

// The arguments of sc_int8_linear_device; strides in elements.
struct Int8Linear {
    const void *x;
    int x_type;
    int64_t x_stride;
    const float *x_scales;      // of an int8 x
    const int8_t *w;
    int64_t w_stride;
    const float *w_scales, *bias;
    int64_t rows, n, k;
    int relu;
    void *y;
    int y_type;
    int64_t y_stride;
    float *y_scales;            // int8 y: a scale for each row, or null
    float output_scale;         // int8 y without y_scales: the one scale
    void *workspace;
    int x_packed, w_packed;     // addresses and strides are multiples of 16 bytes
};

void quantize_tokens(const void *x, int type, int64_t rows, int64_t cols, int64_t x_stride, int8_t *q, int64_t q_stride,
                     float *scales, cudaStream_t s);
void dequantize_tokens(const int8_t *q, int64_t q_stride, const float *scales, float scale, int64_t rows, int64_t cols,
                       void *y, int type, int64_t y_stride, cudaStream_t s);
int64_t int8_linear_workspace(const Int8Linear &p);
// the parts that a call's rows are computed in, see sc_int8_linear_ways
int int8_linear_ways(int64_t rows, int64_t n, int64_t k, bool rows_out, int64_t *out);
void int8_linear(const Int8Linear &p, cudaStream_t s);

}  // namespace sc
