// A teacher's top logits: per row the k largest, their columns and the log-sum-exp, from one read of the row.
//
// The row sits in the shared memory of a cluster (row_slice.cuh).  Pass 1 takes every thread's maximum over
// its elements.  The r-th largest of a CTA's thread maxima, r = ceil(k / parts), has at least r elements of
// the slice at or above it, so the smallest of these over the CTAs has at least k elements of the row at or
// above it: a lower bound for the k-th largest logit, and a close one while there are many more threads
// than r.  Pass 2 sums the exponentials and collects the elements at or above the bound (k and a few more) in
// the first CTA, which ranks them by counting.  Elements are ordered by (value, lower column first) as one
// 64-bit key, so the result does not depend on the order of collection.  Rows with so many elements at
// the bound that the list overflows (ties, rows almost all -inf) find the k-th largest key bit by bit.
#include "../common/host.h"
#include "distill_api.h"
#include "row_slice.cuh"

namespace ttb {
namespace {

using rows::Slice;
namespace cg = cooperative_groups;

constexpr int kCapacity = 1024;  // collected elements

// Monotone whole number of a float: larger for larger values, -0 = +0, NaN above all.
__device__ __forceinline__ uint32_t ordered(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned long long key_of(float v, int col) {
  return (static_cast<unsigned long long>(ordered(v)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(col));
}

// The lowest bit of ordered(v) that values of type T can set (16-bit types widen to floats with zero tails).
template <typename T>
constexpr int lowest_bit() {
  if (std::is_same_v<T, float>) return 0;
  return std::is_same_v<T, __half> ? 13 : 16;
}

struct Shared {
  float max[rows::kMaxParts];
  uint32_t bound[rows::kMaxParts];
  float sum[rows::kMaxParts];
  int count[2][rows::kMaxParts];
  float red[32];
  int redi[32];
  int taken;
};

__device__ __forceinline__ float block_max(float v, float* red) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
  for (int i = 1; i < blockDim.x / 32; ++i) t = fmaxf(t, red[i]);
  __syncthreads();
  return t;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
  for (int i = 1; i < blockDim.x / 32; ++i) t += red[i];
  __syncthreads();
  return t;
}
__device__ __forceinline__ int block_count(int v, int* red) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = red[0];
  for (int i = 1; i < blockDim.x / 32; ++i) t += red[i];
  __syncthreads();
  return t;
}

template <typename T>
__global__ void __launch_bounds__(512) top_logits_kernel(const T* __restrict__ z, long long ldz, int vocab, int k,
                                                         float inv_tau, T* __restrict__ values, int* __restrict__ ids,
                                                         float* __restrict__ lse, int per) {
  constexpr int E = Slice<T>::kVec;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), rank = cluster.block_rank();
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x;
  auto* list = reinterpret_cast<unsigned long long*>(smem + static_cast<size_t>(per) * 16);  // in the first CTA

  const Slice<T> s = rows::start_load(reinterpret_cast<T*>(smem), z + row * ldz, vocab, rank, per);
  if (tid == 0) sh.taken = 0;
  rows::finish_load();
  cluster.sync();  // every CTA of the row runs and has its list empty

  // pass 1: thread maxima (NaN is left out: it enters the list in pass 2 whatever the bound is)
  float mx = -CUDART_INF_F;
  bool any = false;
  for (int v = tid; v < s.nv; v += blockDim.x) {
    float e[E];
    load_vec<E>(s.sm + v * E, e);
#pragma unroll
    for (int i = 0; i < E; ++i) mx = fmaxf(mx, e[i]);
    any = true;
  }
  const uint32_t mine = any ? ordered(mx) : 0u;
  const int r = (k + parts - 1) / parts;
  uint32_t bound = 0;
  for (int bit = 31; bit >= lowest_bit<T>(); --bit) {
    const uint32_t trial = bound | (1u << bit);
    const int c = __syncthreads_count(mine >= trial);
    if (c >= r) bound = trial;
    if (c >= r && c <= r + r / 4) break;  // close enough: a smaller bound only lengthens the list
  }
  const float top = block_max(mx, sh.red);
  if (tid < parts) {
    Shared* peer = cluster.map_shared_rank(&sh, tid);
    peer->max[rank] = top;
    peer->bound[rank] = bound;
  }
  cluster.sync();
  float row_max = -CUDART_INF_F;
  bound = 0xFFFFFFFFu;
  for (int c = 0; c < parts; ++c) {
    row_max = fmaxf(row_max, sh.max[c]);
    bound = min(bound, sh.bound[c]);
  }
  const float ref = isfinite(row_max) ? row_max : 0.f;
  const float least = bound <= ordered(-CUDART_INF_F) ? -CUDART_INF_F : from_ordered(bound);

  // pass 2: sum of exponentials; elements that are not below the bound
  Shared* first = cluster.map_shared_rank(&sh, 0);
  unsigned long long* first_list = cluster.map_shared_rank(list, 0);
  const float c2 = inv_tau * CUDART_L2E_F;
  float sum = 0.f;
  int found = 0;
  for (int v = tid; v < s.nv; v += blockDim.x) {
    float e[E];
    load_vec<E>(s.sm + v * E, e);
    bool some = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      sum += rows::fast_exp2((e[i] - ref) * c2);
      some |= !(e[i] < least);
    }
    if (some) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int col = s.first + v * E + i;
        if (!(e[i] < least) && col >= 0 && col < vocab) {
          ++found;
          const int at = atomicAdd(&first->taken, 1);
          if (at < kCapacity) first_list[at] = key_of(e[i], col);
        }
      }
    }
  }
  sum = block_sum(sum, sh.red);
  found = block_count(found, sh.redi);
  if (tid < parts) {
    Shared* peer = cluster.map_shared_rank(&sh, tid);
    peer->sum[rank] = sum;
    peer->count[0][rank] = found;
  }
  cluster.sync();
  int total = 0;
  for (int c = 0; c < parts; ++c) total += sh.count[0][c];

  if (total > kCapacity) {
    // the k-th largest key, highest bit first; the column's upper bits are ones in every key
    const int col_bits = 32 - __clz(vocab);
    unsigned long long kth = 0;
    int side = 1;
    for (int bit = 63; bit >= 0; --bit) {
      if (bit < 32 && bit >= col_bits) {
        kth |= 1ull << bit;
        continue;
      }
      const unsigned long long trial = kth | (1ull << bit);
      int c = 0;
      for (int v = tid; v < s.nv; v += blockDim.x) {
        float e[E];
        load_vec<E>(s.sm + v * E, e);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int col = s.first + v * E + i;
          c += col >= 0 && col < vocab && key_of(e[i], col) >= trial;
        }
      }
      c = block_count(c, sh.redi);
      if (tid < parts) cluster.map_shared_rank(&sh, tid)->count[side][rank] = c;
      cluster.sync();
      c = 0;
      for (int q = 0; q < parts; ++q) c += sh.count[side][q];
      side ^= 1;
      if (c >= k) kth = trial;
    }
    if (rank == 0 && tid == 0) sh.taken = 0;
    cluster.sync();
    for (int v = tid; v < s.nv; v += blockDim.x) {
      float e[E];
      load_vec<E>(s.sm + v * E, e);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int col = s.first + v * E + i;
        if (col >= 0 && col < vocab && key_of(e[i], col) >= kth) {
          const int at = atomicAdd(&first->taken, 1);
          if (at < kCapacity) first_list[at] = key_of(e[i], col);
        }
      }
    }
    cluster.sync();
    total = k;
  }
  if (rank != 0) return;

  for (int i = tid; i < total; i += blockDim.x) {
    const unsigned long long key = list[i];
    int place = 0;
    for (int j = 0; j < total; ++j) place += list[j] > key;
    if (place < k) {
      values[row * k + place] = from_f32<T>(from_ordered(static_cast<uint32_t>(key >> 32)));
      ids[row * k + place] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
    }
  }
  if (tid == 0) {
    float t = 0.f;
    for (int c = 0; c < parts; ++c) t += sh.sum[c];
    lse[row] = ref * inv_tau + logf(t);
  }
}

}  // namespace

void top_logits(const TopLogitsArgs& a, cudaStream_t stream) {
  TTB_CHECK(a.k >= 1 && a.k <= kTopLogitsMaxK && a.k <= a.vocab, "top logits: k must be between 1 and min(256, columns)");
  TTB_CHECK(logits_row_fits(a.vocab, a.type), "top logits: the rows are too long");
  if (a.rows == 0) return;
  const rows::Plan p = rows::plan_rows(a.rows, a.vocab, scalar_bytes(a.type));
  TTB_CHECK(a.rows * p.parts <= 0x7FFFFFFFLL, "top logits: too many rows");
  const size_t smem = p.slice_bytes + kCapacity * sizeof(unsigned long long);
  with_type(a.type, [&](auto* tz) {
    using T = std::remove_pointer_t<decltype(tz)>;
    auto kernel = top_logits_kernel<T>;
    TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows * p.parts));
    cfg.blockDim = dim3(p.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TTB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(a.z), a.ldz, a.vocab, a.k, a.inv_tau,
                                      static_cast<T*>(a.values), a.ids, a.lse, p.per));
  });
}

}  // namespace ttb
