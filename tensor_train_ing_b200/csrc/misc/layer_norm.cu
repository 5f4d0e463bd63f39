// Layer norm forward and backward (see layer_norm.h for the formulas).
//
// A group of `gw` warps owns one row at a time and keeps it in registers, NV vectors of V elements per
// thread: the row is read once.  The variance is the mean of (x - mu)^2 about the row's own mean
// (two reductions over registers), not E[x^2] - mu^2, which loses all digits of a row whose mean is
// large against its spread.
//
// The backward walks rows with a stride, keeping its columns' dw and db sums in registers; the groups
// of a block add theirs through shared memory in group order and each block writes one row of
// partials, which a second kernel adds in block order: the same inputs give the same bits.
#include "../common/host.h"
#include "../common/vec.cuh"
#include "layer_norm.h"

namespace ttb {
namespace {

constexpr int kThreads = 512;

// Sum over the row group's threads; `slot` alternates between two halves of `red` so that one barrier
// per sum is enough.
__device__ __forceinline__ float2 group_sum2(float a, float b, float2* red, int warp, int first, int gw, int bar) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (gw == 1) return make_float2(a, b);
  if ((threadIdx.x & 31) == 0) red[warp] = make_float2(a, b);
  named_barrier(bar, gw * 32);
  float2 t = red[first];
  for (int i = 1; i < gw; ++i) {
    const float2 u = red[first + i];
    t.x += u.x;
    t.y += u.y;
  }
  return t;
}

template <typename TX, typename TY, int V, int NV>
__global__ void __launch_bounds__(kThreads) layer_norm_fwd_kernel(const TX* __restrict__ x, long long ldx,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ b, TY* __restrict__ y,
                                                                 float* __restrict__ mean, float* __restrict__ rstd,
                                                                 long long rows, int d, float eps, int gw) {
  __shared__ float2 red[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / gw, groups = kThreads / 32 / gw;
  const int t = (warp - group * gw) * 32 + lane;
  const int step = gw * 32 * V;
  const float inv_d = 1.f / d;
  for (long long row = static_cast<long long>(blockIdx.x) * groups + group; row < rows;
       row += static_cast<long long>(gridDim.x) * groups) {
    const TX* xr = x + row * ldx;
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (j < d) {
        load_vec<V>(xr + j, v[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[i][k];
      }
    }
    const float mu = group_sum2(s, 0.f, red[0], warp, group * gw, gw, 1 + group).x * inv_d;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * step + t * V < d) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          v[i][k] -= mu;
          q += v[i][k] * v[i][k];
        }
      }
    }
    const float var = group_sum2(q, 0.f, red[1], warp, group * gw, gw, 1 + group).x * inv_d;
    const float r = 1.f / sqrtf(var + eps);
    if (mean != nullptr && t == 0) {
      mean[row] = mu;
      rstd[row] = r;
    }
    TY* yr = y + row * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (j < d) {
        float wv[V], o[V];
        load_vec<V>(w + j, wv);
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = v[i][k] * r * wv[k];
        if (b != nullptr) {
          float bv[V];
          load_vec<V>(b + j, bv);
#pragma unroll
          for (int k = 0; k < V; ++k) o[k] += bv[k];
        }
        store_vec<V>(yr + j, o);
      }
    }
  }
}

template <typename TX, typename TY, int V, int NV>
__global__ void __launch_bounds__(kThreads) layer_norm_bwd_kernel(
    const TY* __restrict__ dy, long long lddy, const TX* __restrict__ x, long long ldx, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, TX* __restrict__ dx, float* __restrict__ partials,
    long long rows, int d, int gw) {
  extern __shared__ float acc[];  // 2 d floats: the block's dw and db
  __shared__ float2 red[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / gw, groups = kThreads / 32 / gw;
  const int t = (warp - group * gw) * 32 + lane;
  const int step = gw * 32 * V;
  const float inv_d = 1.f / d;
  float wv[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = i * step + t * V;
    if (j < d) load_vec<V>(w + j, wv[i]);
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.f;
  }
  int it = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * groups + group; row < rows;
       row += static_cast<long long>(gridDim.x) * groups, it ^= 1) {
    const TX* xr = x + row * ldx;
    const TY* dyr = dy + row * lddy;
    const float mu = mean[row], r = rstd[row];
    float xh[NV][V], g[NV][V];
    float sa = 0.f, sb = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (j < d) {
        load_vec<V>(xr + j, xh[i]);
        load_vec<V>(dyr + j, g[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * step + t * V < d) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          xh[i][k] = (xh[i][k] - mu) * r;
          dw[i][k] += g[i][k] * xh[i][k];
          db[i][k] += g[i][k];
          g[i][k] *= wv[i][k];
          sa += g[i][k];
          sb += g[i][k] * xh[i][k];
        }
      }
    }
    const float2 sum = group_sum2(sa, sb, red[it], warp, group * gw, gw, 1 + group);
    const float ma = sum.x * inv_d, mb = sum.y * inv_d;
    TX* dxr = dx + row * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (j < d) {
        float o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = r * (g[i][k] - ma - xh[i][k] * mb);
        store_vec<V>(dxr + j, o);
      }
    }
  }
  for (int q = 0; q < groups; ++q) {
    if (q > 0) __syncthreads();
    if (q != group) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (j < d) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          acc[j + k] = (q > 0 ? acc[j + k] : 0.f) + dw[i][k];
          acc[d + j + k] = (q > 0 ? acc[d + j + k] : 0.f) + db[i][k];
        }
      }
    }
  }
  __syncthreads();
  float* out = partials + static_cast<long long>(blockIdx.x) * 2 * d;
  for (int j = threadIdx.x; j < 2 * d; j += blockDim.x) out[j] = acc[j];
}

// dw | db [j] = sum over the partial rows in a fixed order: 32 columns x 8 row classes per block.
__global__ void __launch_bounds__(256) layer_norm_param_grad_kernel(const float* __restrict__ partials, int count,
                                                                    int d, float* __restrict__ dw,
                                                                    float* __restrict__ db) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x % 32, c = threadIdx.x / 32;
  const int j = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (j < 2 * d)
    for (int p = c; p < count; p += 8) s += partials[static_cast<long long>(p) * 2 * d + j];
  red[c][lane] = s;
  __syncthreads();
  if (c == 0 && j < 2 * d) {
    float t = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) t += red[q][lane];
    if (j < d)
      dw[j] = t;
    else if (db != nullptr)
      db[j - d] = t;
  }
}

// How a row is spread: `gw` warps per row (a power of two), NV vectors of V elements per thread.
struct Split {
  int v, nv, gw, groups;
};

constexpr int kPerThread = 16;  // elements of a row a thread holds, up to d = 8192 (twice that beyond)

Split split_row(int d, int v) {
  int gw = 1;
  while (gw < kThreads / 32 && gw * 32 * kPerThread < d) gw *= 2;
  Split s;
  s.v = v;
  s.gw = gw;
  s.nv = (d + gw * 32 * v - 1) / (gw * 32 * v);
  s.groups = kThreads / 32 / gw;
  return s;
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename F>
void with_split(const Split& s, F&& f) {
  using std::integral_constant;
  if (s.v == 4) {
    if (s.nv == 1) return f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (s.nv == 2) return f(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    if (s.nv == 3) return f(integral_constant<int, 4>{}, integral_constant<int, 3>{});
    if (s.nv == 4) return f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    return f(integral_constant<int, 4>{}, integral_constant<int, 8>{});
  }
  if (s.nv <= 4) return f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  if (s.nv <= 8) return f(integral_constant<int, 1>{}, integral_constant<int, 8>{});
  if (s.nv <= 16) return f(integral_constant<int, 1>{}, integral_constant<int, 16>{});
  return f(integral_constant<int, 1>{}, integral_constant<int, 32>{});
}

void check(const LayerNormShape& s) {
  TTB_CHECK(s.d >= 1 && s.d <= kLayerNormMaxDim, "layer norm: the last dimension must be between 1 and 16384");
}

int blocks_for(const LayerNormShape& s, const Split& sp, int per_sm) {
  const long long need = (s.rows + sp.groups - 1) / sp.groups;
  const long long most = static_cast<long long>(num_sms()) * per_sm;
  return static_cast<int>(need < most ? need : most);
}

}  // namespace

void layer_norm_fwd(const LayerNormShape& s, const void* x, long long ldx, const float* w, const float* b, void* y,
                    float* mean, float* rstd, float eps, cudaStream_t stream) {
  check(s);
  if (s.rows == 0) return;
  const bool vec = s.d % 4 == 0 && ldx % 4 == 0 && aligned(x, 4 * scalar_bytes(s.x)) &&
                   aligned(y, 4 * scalar_bytes(s.y)) && aligned(w, 16) && (b == nullptr || aligned(b, 16));
  const Split sp = split_row(s.d, vec ? 4 : 1);
  with_type(s.x, [&](auto* tx) {
    using TX = std::remove_pointer_t<decltype(tx)>;
    with_type(s.y, [&](auto* ty) {
      using TY = std::remove_pointer_t<decltype(ty)>;
      with_split(sp, [&](auto v, auto nv) {
        layer_norm_fwd_kernel<TX, TY, decltype(v)::value, decltype(nv)::value>
            <<<blocks_for(s, sp, 4), kThreads, 0, stream>>>(static_cast<const TX*>(x), ldx, w, b, static_cast<TY*>(y),
                                                           mean, rstd, s.rows, s.d, eps, sp.gw);
      });
    });
  });
  TTB_CUDA_CHECK(cudaGetLastError());
}

int layer_norm_bwd_partials(const LayerNormShape& s) {
  check(s);
  return blocks_for(s, split_row(s.d, 4), 1);
}

void layer_norm_bwd(const LayerNormShape& s, const void* dy, long long lddy, const void* x, long long ldx,
                    const float* w, const float* mean, const float* rstd, void* dx, float* dw, float* db,
                    float* partials, cudaStream_t stream) {
  check(s);
  TTB_CHECK(s.rows > 0, "layer norm backward: no rows");
  const bool vec = s.d % 4 == 0 && ldx % 4 == 0 && lddy % 4 == 0 && aligned(x, 4 * scalar_bytes(s.x)) &&
                   aligned(dx, 4 * scalar_bytes(s.x)) && aligned(dy, 4 * scalar_bytes(s.y)) && aligned(w, 16);
  const Split sp = split_row(s.d, vec ? 4 : 1);
  const int grid = layer_norm_bwd_partials(s);
  const size_t smem = static_cast<size_t>(s.d) * 2 * sizeof(float);
  with_type(s.x, [&](auto* tx) {
    using TX = std::remove_pointer_t<decltype(tx)>;
    with_type(s.y, [&](auto* ty) {
      using TY = std::remove_pointer_t<decltype(ty)>;
      with_split(sp, [&](auto v, auto nv) {
        auto kernel = layer_norm_bwd_kernel<TX, TY, decltype(v)::value, decltype(nv)::value>;
        if (smem > 40 * 1024)
          TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              static_cast<int>(smem)));
        kernel<<<grid, kThreads, smem, stream>>>(static_cast<const TY*>(dy), lddy, static_cast<const TX*>(x), ldx, w,
                                                mean, rstd, static_cast<TX*>(dx), partials, s.rows, s.d, sp.gw);
      });
    });
  });
  TTB_CUDA_CHECK(cudaGetLastError());
  layer_norm_param_grad_kernel<<<(2 * s.d + 31) / 32, 256, 0, stream>>>(partials, grid, s.d, dw, db);
  TTB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace ttb
