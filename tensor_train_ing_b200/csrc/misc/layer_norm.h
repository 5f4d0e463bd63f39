// Layer norm over the last dimension, forward and backward:
//
//   mu = mean_j x,  rstd = 1 / sqrt(mean_j (x - mu)^2 + eps),  xhat = (x - mu) rstd,  y = xhat w + b
//   g = dy w,  dx = rstd (g - mean_j g - xhat mean_j (g xhat)),  dw = sum_n dy xhat,  db = sum_n dy
//
// x and y are fp32, bf16 or fp16 rows (dy has y's type, dx x's); w, b and every sum are fp32.
#pragma once

#include <cuda_runtime.h>

#include "../common/dtype.h"

namespace ttb {

constexpr int kLayerNormMaxDim = 16384;

struct LayerNormShape {
  long long rows;
  int d;
  ScalarType x, y;
};

// x: rows `ldx` elements apart; y: dense rows.  mean / rstd (fp32 per row) may both be null.  b may be null.
void layer_norm_fwd(const LayerNormShape& s, const void* x, long long ldx, const float* w, const float* b, void* y,
                    float* mean, float* rstd, float eps, cudaStream_t stream);

// Rows of the backward's partial sums (each 2 d floats) for this shape and these pointers.
int layer_norm_bwd_partials(const LayerNormShape& s);

// dy: rows `lddy` apart; dx: dense rows; dw, db: [d] fp32, written (db may be null); partials: fp32 scratch of
// layer_norm_bwd_partials(s) * 2 d.
void layer_norm_bwd(const LayerNormShape& s, const void* dy, long long lddy, const void* x, long long ldx,
                    const float* w, const float* mean, const float* rstd, void* dx, float* dw, float* db,
                    float* partials, cudaStream_t stream);

}  // namespace ttb
