// Layer norm forward and backward (see layer_norm.h for the formulas).
//
// A group of `gw` warps owns one row at a time and keeps it in registers, NV vectors of V elements per
// thread: the row is read once.  The variance is the mean of (x - mu)^2 about the row's own mean
// (two reductions over registers), not E[x^2] - mu^2, which loses all digits of a row whose mean is
// large against its spread.
//
// Rows that can be copied in 16-byte pieces arrive through a ring of shared-memory slots that every group fills ahead
// with bulk copies (one barrier per slot): an SM keeps up to about 200 KB of loads under way whatever the
// register file allows.  A slot is filled again right after the group's barrier of its row, at which every
// thread has taken its part.  Other rows are loaded straight into registers, those of odd width an element per lane and
// access, which bounds them: 3001 rows of 1037 fp32 columns take 29 us (4 us for the bytes), with backward 53 us (10 us).
//
// The backward walks rows with a stride, keeping its columns' dw and db sums in registers; the groups
// of a block add theirs through shared memory in group order and each block writes one row of
// partials, which a second kernel adds in block order: the same inputs give the same bits.
#include "../common/host.h"
#include "../common/sm100.cuh"
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

__device__ __forceinline__ float group_sum(float a, float* red, int warp, int first, int gw, int bar) {
  a = warp_sum(a);
  if (gw == 1) return a;
  if ((threadIdx.x & 31) == 0) red[warp] = a;
  named_barrier(bar, gw * 32);
  float t = red[first];
  for (int i = 1; i < gw; ++i) t += red[first + i];
  return t;
}

template <typename TX, typename TY, int V, int NV>
__global__ void __launch_bounds__(kThreads) layer_norm_fwd_kernel(const TX* __restrict__ x, long long ldx,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ b, TY* __restrict__ y,
                                                                 float* __restrict__ mean, float* __restrict__ rstd,
                                                                 long long rows, int d, float eps, int gw) {
  __shared__ float red[2][kThreads / 32];
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
    const float mu = group_sum(s, red[0], warp, group * gw, gw, 1 + group) * inv_d;
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
    const float var = group_sum(q, red[1], warp, group * gw, gw, 1 + group) * inv_d;
    const float r = rsqrtf(var + eps);
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

// The block's row of partials: its groups' dw and db, added in group order.
template <int V, int NV>
__device__ __forceinline__ void write_partials(float* acc, const float (&dw)[NV][V], const float (&db)[NV][V],
                                               float* __restrict__ partials, int d, int t, int step, int group,
                                               int groups) {
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
  write_partials<V, NV>(acc, dw, db, partials, d, t, step, group, groups);
}

// ---------------------------------------------------------------------------------------------
// The same with rows arriving through the ring.
constexpr int kMaxSlots = 8;

// Elements of a row a thread holds.  What a warp does once per row (sums across lanes and warps, waiting for the slot)
// costs as much as about 20 elements per lane, so few warps with much of a row each beat many with little.  16384 rows
// of 2048 fp32 columns to bf16 (bytes alone: 31 us): the forward took 61 us with 8 elements a thread, 46 us with 32 and 41 us
// with 64.  The backward also holds its columns' sums of dw and db, so 128 registers end at 24 elements: 78 us with
// 8, 66 us with 16, 61 us with 24 (51 us for its bytes); 8192 rows of 6144 bf16 columns 81 us (46 us).  It is bound by each
// row's chain of loads, sums across warps and stores, of which an SM has two (6144 columns) or four (2048) under way.
constexpr int kFwdPerThread = 64, kBwdPerThread = 24;
constexpr int kFwdBlocks = 1, kBwdBlocks = 1;  // of 512 threads that fit an SM then

struct Ring {
  int slots;        // per group
  int x_bytes;      // of a row; the slot's second row follows (backward)
  int slot_bytes;
  uint32_t* status;
};

// One group's side of its ring: waits are bounded, and one that runs out is reported and waited for once more so that
// the copy does not outlive the block.
struct RingSide {
  uint64_t* full;  // [slots]
  uint8_t* base;
  int slot, phase;
  __device__ __forceinline__ const uint8_t* wait(const Ring& r) {
    if (!mbar_wait(&full[slot], phase, r.status, kErrTimeoutProducer))
      mbar_wait(&full[slot], phase, r.status, kErrTimeoutProducer);
    return base + slot * r.slot_bytes;
  }
  __device__ __forceinline__ void next(const Ring& r) {
    if (++slot == r.slots) {
      slot = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ RingSide ring_side(const Ring& r, uint64_t (*full)[kMaxSlots], uint8_t* smem, int group,
                                              int groups) {
  if (threadIdx.x == 0) {
    for (int g = 0; g < groups; ++g)
      for (int i = 0; i < r.slots; ++i) mbar_init(&full[g][i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  return RingSide{full[group], smem + static_cast<size_t>(group) * r.slots * r.slot_bytes, 0, 0};
}

template <typename TX, typename TY, int V, int NV, int SURE>
__global__ void __launch_bounds__(kThreads, kFwdBlocks) layer_norm_fwd_ring_kernel(
    const TX* __restrict__ x, long long ldx, const float* __restrict__ w, const float* __restrict__ b,
    TY* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, long long rows, int d, float eps, int gw,
    const __grid_constant__ Ring ring) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t full[kThreads / 32][kMaxSlots];
  __shared__ float red[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / gw, groups = kThreads / 32 / gw;
  const int t = (warp - group * gw) * 32 + lane;
  const int step = gw * 32 * V;
  const float inv_d = 1.f / d;
  const long long stride = static_cast<long long>(gridDim.x) * groups;
  long long row = static_cast<long long>(blockIdx.x) * groups + group;
  RingSide side = ring_side(ring, full, smem, group, groups);
  const auto fill = [&](int slot, long long r) {
    mbar_arrive_expect_tx(&side.full[slot], ring.x_bytes);
    bulk_load(side.base + slot * ring.slot_bytes, x + r * ldx, ring.x_bytes, &side.full[slot]);
  };
  if (t == 0)
    for (int i = 0; i < ring.slots && row + i * stride < rows; ++i) fill(i, row + i * stride);
  for (; row < rows; row += stride) {
    const TX* xr = reinterpret_cast<const TX*>(side.wait(ring));
    float v[NV][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (i < SURE || j < d) {
        load_vec<V>(xr + j, v[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[i][k];
      }
    }
    const float mu = group_sum(s, red[0], warp, group * gw, gw, 1 + group) * inv_d;
    if (gw == 1) __syncwarp();
    if (t == 0 && row + ring.slots * stride < rows) fill(side.slot, row + ring.slots * stride);
    side.next(ring);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i < SURE || i * step + t * V < d) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          v[i][k] -= mu;
          q += v[i][k] * v[i][k];
        }
      }
    }
    const float var = group_sum(q, red[1], warp, group * gw, gw, 1 + group) * inv_d;
    const float r = rsqrtf(var + eps);
    if (mean != nullptr && t == 0) {
      mean[row] = mu;
      rstd[row] = r;
    }
    TY* yr = y + row * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (i < SURE || j < d) {
        float wv[V], o[V];
        load_vec<V>(w + j, wv);
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = v[i][k] * r * wv[k];
        if (b != nullptr) {
          load_vec<V>(b + j, wv);
#pragma unroll
          for (int k = 0; k < V; ++k) o[k] += wv[k];
        }
        store_vec<V>(yr + j, o);
      }
    }
  }
}

template <typename TX, typename TY, int V, int NV, int SURE>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) layer_norm_bwd_ring_kernel(
    const TY* __restrict__ dy, long long lddy, const TX* __restrict__ x, long long ldx, const float* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, TX* __restrict__ dx, float* __restrict__ partials,
    long long rows, int d, int gw, const __grid_constant__ Ring ring) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t full[kThreads / 32][kMaxSlots];
  __shared__ float2 red[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp / gw, groups = kThreads / 32 / gw;
  const int t = (warp - group * gw) * 32 + lane;
  const int step = gw * 32 * V;
  const float inv_d = 1.f / d;
  const long long stride = static_cast<long long>(gridDim.x) * groups;
  long long row = static_cast<long long>(blockIdx.x) * groups + group;
  RingSide side = ring_side(ring, full, smem, group, groups);
  const int dy_bytes = ring.slot_bytes - ring.x_bytes;
  const auto fill = [&](int slot, long long r) {
    uint8_t* to = side.base + slot * ring.slot_bytes;
    mbar_arrive_expect_tx(&side.full[slot], ring.slot_bytes);
    bulk_load(to, x + r * ldx, ring.x_bytes, &side.full[slot]);
    bulk_load(to + ring.x_bytes, dy + r * lddy, dy_bytes, &side.full[slot]);
  };
  if (t == 0)
    for (int i = 0; i < ring.slots && row + i * stride < rows; ++i) fill(i, row + i * stride);
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.f;
  float mu = row < rows ? mean[row] : 0.f, r = row < rows ? rstd[row] : 0.f;
  for (int it = 0; row < rows; row += stride, it ^= 1) {
    const long long after = row + stride < rows ? row + stride : row;
    const float mu_after = mean[after], r_after = rstd[after];
    const TX* xr = reinterpret_cast<const TX*>(side.wait(ring));
    const TY* dyr = reinterpret_cast<const TY*>(reinterpret_cast<const uint8_t*>(xr) + ring.x_bytes);
    float xh[NV][V], g[NV][V];
    float sa = 0.f, sb = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (i < SURE || j < d) {
        float wv[V];
        load_vec<V>(xr + j, xh[i]);
        load_vec<V>(dyr + j, g[i]);
        load_vec<V>(w + j, wv);  // from L1: the registers hold the sums
#pragma unroll
        for (int k = 0; k < V; ++k) {
          xh[i][k] = (xh[i][k] - mu) * r;
          dw[i][k] += g[i][k] * xh[i][k];
          db[i][k] += g[i][k];
          g[i][k] *= wv[k];
          sa += g[i][k];
          sb += g[i][k] * xh[i][k];
        }
      }
    }
    const float2 sum = group_sum2(sa, sb, red[it], warp, group * gw, gw, 1 + group);
    if (gw == 1) __syncwarp();
    if (t == 0 && row + ring.slots * stride < rows) fill(side.slot, row + ring.slots * stride);
    side.next(ring);
    const float ma = sum.x * inv_d, mb = sum.y * inv_d;
    TX* dxr = dx + row * d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * step + t * V;
      if (i < SURE || j < d) {
        float o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = r * (g[i][k] - ma - xh[i][k] * mb);
        store_vec<V>(dxr + j, o);
      }
    }
    mu = mu_after;
    r = r_after;
  }
  __syncthreads();  // every group is done with its slots: their memory takes the sums
  write_partials<V, NV>(reinterpret_cast<float*>(smem), dw, db, partials, d, t, step, group, groups);
}

// dw | db [j] = sum over the partial rows in a fixed order: 32 columns x 32 row classes per block.
__global__ void __launch_bounds__(1024) layer_norm_param_grad_kernel(const float* __restrict__ partials, int count,
                                                                     int d, float* __restrict__ dw,
                                                                     float* __restrict__ db) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x % 32, c = threadIdx.x / 32;
  const int j = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (j < 2 * d) {
#pragma unroll 4
    for (int p = c; p < count; p += 32) s += partials[static_cast<long long>(p) * 2 * d + j];
  }
  red[c][lane] = s;
  __syncthreads();
  const float t = warp_sum(red[lane][c]);  // warp c: column c of the block
  const int column = blockIdx.x * 32 + c;
  if (lane == 0 && column < 2 * d) {
    if (column < d)
      dw[column] = t;
    else if (db != nullptr)
      db[column - d] = t;
  }
}

// How a row is spread: `gw` warps per row (a power of two), NV vectors of V elements per thread.
struct Split {
  int v, nv, gw, groups;
};

// `most`: elements of a row a thread holds, while 16 warps suffice for that.
Split split_row(int d, int v, int most) {
  int gw = 1;
  while (gw < kThreads / 32 && gw * 32 * most < d) gw *= 2;
  Split s;
  s.v = v;
  s.gw = gw;
  s.nv = (d + gw * 32 * v - 1) / (gw * 32 * v);
  s.groups = kThreads / 32 / gw;
  return s;
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// f(V, NV, SURE) with the smallest listed NV >= nv; SURE is the one before it: every thread has that many vectors.
template <int V, int BEFORE, int FIRST, int... REST, typename F>
void with_vectors(int nv, F&& f) {
  using std::integral_constant;
  if (nv <= FIRST) return f(integral_constant<int, V>{}, integral_constant<int, FIRST>{}, integral_constant<int, BEFORE>{});
  if constexpr (sizeof...(REST) > 0) return with_vectors<V, FIRST, REST...>(nv, f);
  TTB_CHECK(false, "layer norm: row split");
}
template <typename F>
void with_split(const Split& s, F&& f) {  // rows straight into registers
  if (s.v == 4) return with_vectors<4, 0, 1, 2, 4, 8>(s.nv, f);
  with_vectors<1, 0, 4, 8, 16, 32>(s.nv, f);
}
template <typename F>
void with_fwd_ring_split(const Split& s, F&& f) {
  if (s.v == 8) return with_vectors<8, 0, 1, 2, 4, 6, 8>(s.nv, f);
  with_vectors<4, 0, 1, 2, 4, 8, 12, 16>(s.nv, f);
}
template <typename F>
void with_bwd_ring_split(const Split& s, F&& f) {
  if (s.v == 8) return with_vectors<8, 0, 1, 2, 3, 4>(s.nv, f);
  with_vectors<4, 0, 1, 2, 3, 4, 6, 8>(s.nv, f);
}

// Whether rows of d elements, ld apart, can be copied in 16-byte pieces.
bool whole_rows(const void* p, long long ld, int d, ScalarType t) {
  const int b = scalar_bytes(t);
  return aligned(p, 16) && (ld * b) % 16 == 0 && (static_cast<long long>(d) * b) % 16 == 0;
}

// 16-byte shared-memory reads of the wider type.
Split ring_split(const LayerNormShape& s, int most) {
  return split_row(s.d, s.x == ScalarType::kF32 || s.y == ScalarType::kF32 ? 4 : 8, most);
}
Ring make_ring(const Split& sp, int x_bytes, int slot_bytes, int blocks_per_sm, size_t at_least, size_t& smem) {
  const size_t budget = 208 * 1024 / blocks_per_sm;
  Ring r;
  r.x_bytes = x_bytes;
  r.slot_bytes = slot_bytes;
  const long long fit = static_cast<long long>(budget / (static_cast<size_t>(sp.groups) * slot_bytes));
  r.slots = static_cast<int>(fit < 1 ? 1 : fit > kMaxSlots ? kMaxSlots : fit);
  r.status = status_ptr();
  smem = static_cast<size_t>(sp.groups) * r.slots * slot_bytes;
  if (smem < at_least) smem = at_least;
  return r;
}

void check(const LayerNormShape& s) {
  TTB_CHECK(s.d >= 1 && s.d <= kLayerNormMaxDim, "layer norm: the last dimension must be between 1 and 16384");
}

int blocks_for(const LayerNormShape& s, const Split& sp, int per_sm) {
  const long long need = (s.rows + sp.groups - 1) / sp.groups;
  const long long most = static_cast<long long>(num_sms()) * per_sm;
  return static_cast<int>(need < most ? need : most);
}

// The ring kernels are built for the pairs of types that models use: fp32 rows to any type, 16-bit rows to their own.
bool ring_types(const LayerNormShape& s) { return s.x == ScalarType::kF32 || s.x == s.y; }
template <typename F>
void with_ring_types(const LayerNormShape& s, F&& f) {
  if (s.x == ScalarType::kF32) return with_type(s.y, [&](auto* ty) { f(static_cast<float*>(nullptr), ty); });
  with_type(s.x, [&](auto* tx) {
    if constexpr (!std::is_same_v<decltype(tx), float*>) f(tx, tx);
  });
}
template <typename F>
void with_types(const LayerNormShape& s, F&& f) {
  with_type(s.x, [&](auto* tx) { with_type(s.y, [&](auto* ty) { f(tx, ty); }); });
}

}  // namespace

void layer_norm_fwd(const LayerNormShape& s, const void* x, long long ldx, const float* w, const float* b, void* y,
                    float* mean, float* rstd, float eps, cudaStream_t stream) {
  check(s);
  if (s.rows == 0) return;
  if (ring_types(s) && whole_rows(x, ldx, s.d, s.x) && s.d % 8 == 0 && aligned(y, 16) && aligned(w, 16) && aligned(b, 16)) {
    const Split sp = ring_split(s, kFwdPerThread);
    size_t smem;
    const int bytes = s.d * scalar_bytes(s.x);
    const Ring ring = make_ring(sp, bytes, bytes, kFwdBlocks, 0, smem);
    with_ring_types(s, [&](auto* tx, auto* ty) {
      using TX = std::remove_pointer_t<decltype(tx)>;
      using TY = std::remove_pointer_t<decltype(ty)>;
      with_fwd_ring_split(sp, [&](auto v, auto nv, auto sure) {
        auto kernel = layer_norm_fwd_ring_kernel<TX, TY, decltype(v)::value, decltype(nv)::value, decltype(sure)::value>;
        TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        kernel<<<blocks_for(s, sp, kFwdBlocks), kThreads, smem, stream>>>(
            static_cast<const TX*>(x), ldx, w, b, static_cast<TY*>(y), mean, rstd, s.rows, s.d, eps, sp.gw, ring);
      });
    });
    TTB_CUDA_CHECK(cudaGetLastError());
    return;
  }
  const bool vec = s.d % 4 == 0 && ldx % 4 == 0 && aligned(x, 4 * scalar_bytes(s.x)) &&
                   aligned(y, 4 * scalar_bytes(s.y)) && aligned(w, 16) && aligned(b, 16);
  const Split sp = split_row(s.d, vec ? 4 : 1, 16);
  with_types(s, [&](auto* tx, auto* ty) {
    using TX = std::remove_pointer_t<decltype(tx)>;
    using TY = std::remove_pointer_t<decltype(ty)>;
    with_split(sp, [&](auto v, auto nv, auto) {
      layer_norm_fwd_kernel<TX, TY, decltype(v)::value, decltype(nv)::value>
          <<<blocks_for(s, sp, 4), kThreads, 0, stream>>>(static_cast<const TX*>(x), ldx, w, b, static_cast<TY*>(y),
                                                          mean, rstd, s.rows, s.d, eps, sp.gw);
    });
  });
  TTB_CUDA_CHECK(cudaGetLastError());
}

int layer_norm_bwd_partials(const LayerNormShape& s) {
  check(s);
  const int ring = blocks_for(s, ring_split(s, kBwdPerThread), kBwdBlocks), plain = blocks_for(s, split_row(s.d, 4, 16), 1);
  return ring > plain ? ring : plain;
}

void layer_norm_bwd(const LayerNormShape& s, const void* dy, long long lddy, const void* x, long long ldx,
                    const float* w, const float* mean, const float* rstd, void* dx, float* dw, float* db,
                    float* partials, cudaStream_t stream) {
  check(s);
  TTB_CHECK(s.rows > 0, "layer norm backward: no rows");
  const size_t sums = static_cast<size_t>(s.d) * 2 * sizeof(float);
  int grid = 0;
  if (ring_types(s) && whole_rows(x, ldx, s.d, s.x) && whole_rows(dy, lddy, s.d, s.y) && s.d % 8 == 0 && aligned(dx, 16) &&
      aligned(w, 16)) {
    const Split sp = ring_split(s, kBwdPerThread);
    size_t smem;
    const int bytes = s.d * scalar_bytes(s.x);
    const Ring ring = make_ring(sp, bytes, bytes + s.d * scalar_bytes(s.y), kBwdBlocks, sums, smem);
    grid = blocks_for(s, sp, kBwdBlocks);
    with_ring_types(s, [&](auto* tx, auto* ty) {
      using TX = std::remove_pointer_t<decltype(tx)>;
      using TY = std::remove_pointer_t<decltype(ty)>;
      with_bwd_ring_split(sp, [&](auto v, auto nv, auto sure) {
        auto kernel = layer_norm_bwd_ring_kernel<TX, TY, decltype(v)::value, decltype(nv)::value, decltype(sure)::value>;
        TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        kernel<<<grid, kThreads, smem, stream>>>(static_cast<const TY*>(dy), lddy, static_cast<const TX*>(x), ldx, w,
                                                 mean, rstd, static_cast<TX*>(dx), partials, s.rows, s.d, sp.gw, ring);
      });
    });
  } else {
    const bool vec = s.d % 4 == 0 && ldx % 4 == 0 && lddy % 4 == 0 && aligned(x, 4 * scalar_bytes(s.x)) &&
                     aligned(dx, 4 * scalar_bytes(s.x)) && aligned(dy, 4 * scalar_bytes(s.y)) && aligned(w, 16);
    const Split sp = split_row(s.d, vec ? 4 : 1, 16);
    grid = blocks_for(s, sp, 1);
    with_types(s, [&](auto* tx, auto* ty) {
      using TX = std::remove_pointer_t<decltype(tx)>;
      using TY = std::remove_pointer_t<decltype(ty)>;
      with_split(sp, [&](auto v, auto nv, auto) {
        auto kernel = layer_norm_bwd_kernel<TX, TY, decltype(v)::value, decltype(nv)::value>;
        if (sums > 40 * 1024)
          TTB_CUDA_CHECK(
              cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sums)));
        kernel<<<grid, kThreads, sums, stream>>>(static_cast<const TY*>(dy), lddy, static_cast<const TX*>(x), ldx, w,
                                                 mean, rstd, static_cast<TX*>(dx), partials, s.rows, s.d, sp.gw);
      });
    });
  }
  TTB_CUDA_CHECK(cudaGetLastError());
  layer_norm_param_grad_kernel<<<(2 * s.d + 31) / 32, 1024, 0, stream>>>(partials, grid, s.d, dw, db);
  TTB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace ttb
