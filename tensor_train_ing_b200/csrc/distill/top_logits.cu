// A teacher's top logits: per row the k largest, their columns and the log-sum-exp, from one read of the row.
//
// The row sits in the shared memory of a cluster, usually of one CTA (row_slice.cuh).  As it arrives every thread takes the
// maximum of its elements.  The r-th largest of a CTA's thread maxima, r = ceil(k / parts), has at least r
// elements of the slice at or above it, so the smallest of these over the CTAs has at least k elements of the row
// at or above it: a lower bound for the k-th largest logit, and a close one while there are many more
// threads than r.  Only threads whose maximum reaches the bound can hold such elements: their vectors (about k
// threads') are looked through once more, one vector per lane, and the elements found (k and a few more)
// are ranked by counting in the first CTA.  Elements are ordered by (value, lower column first) as one
// 64-bit key, so the result does not depend on the order of collection.  Rows with so many elements at the bound that
// the list overflows (ties, rows almost all -inf), and rows with NaN, find the k-th largest key bit by bit.
//
// Few rows, and rows shorter than the persistent kernel's.  Latency bounds it: the copy, the maxima, the bound and the ranking
// follow one another, and only the other CTAs of the SM fill the gaps.  4 rows of 50257 fp32 logits, the top 32: 12 us with the
// launch; 8288 rows of 32768 bf16, the top 8: 149 us (83 us for the bytes).
#include "../common/host.h"
#include "top_common.cuh"

namespace ttb {
namespace {

using rows::Slice;
namespace cg = cooperative_groups;
using namespace top;

struct Shared {
  uint64_t bars[rows::kStages];
  uint32_t maxima[rows::kMaxThreads];  // ordered() of the thread maxima
  unsigned short hit[rows::kMaxThreads];
  uint32_t warp_max[rows::kMaxThreads / 32];
  float warp_sums[rows::kMaxThreads / 32];
  int red[rows::kMaxThreads / 32];
  uint32_t bound[rows::kMaxParts];
  rows::Ref ref[rows::kMaxParts];
  float sum[rows::kMaxParts];
  int count[2][rows::kMaxParts];
  int hits, taken;
};

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
__global__ void __launch_bounds__(rows::kMaxThreads) top_logits_kernel(const T* __restrict__ z, long long ldz,
                                                                      int vocab, int k, float inv_tau,
                                                                      T* __restrict__ values, int* __restrict__ ids,
                                                                      float* __restrict__ lse, int per, int parts,
                                                                      uint32_t* status) {
  constexpr int E = Slice<T>::kVec;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = parts > 1 ? cluster.block_rank() : 0;
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  auto* list = reinterpret_cast<unsigned long long*>(smem + static_cast<size_t>(per) * 16);  // in the first CTA

  if (tid == 0) sh.hits = sh.taken = 0;
  const Slice<T> s = rows::start_load(reinterpret_cast<T*>(smem), sh.bars, z + row * ldz, vocab, rank, per);
  if (parts > 1) cluster.barrier_arrive();  // this CTA runs and its counters are set

  // Thread maxima.  NaN is left out here; it shows in the sum.
  const float mx = rows::max_while_loading(s, sh.bars, status);
  const uint32_t mine = tid < s.nv ? ordered(mx) : 0u;
  sh.maxima[tid] = mine;
  uint32_t top = __reduce_max_sync(0xffffffffu, mine);
  if (lane == 0) sh.warp_max[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? sh.warp_max[lane] : 0u);
  const float c = inv_tau * CUDART_L2E_F;
  const rows::Ref ref(top == 0u ? -CUDART_INF_F : from_ordered(top), c);
  if (parts > 1) cluster.barrier_wait();
  if (warp == 0) {
    const uint32_t bound = find_bound<T>(sh.maxima, blockDim.x, (k + parts - 1) / parts);
    if (lane < parts) (parts > 1 ? cluster.map_shared_rank(&sh, lane) : &sh)->bound[rank] = bound;
  }

  // sum of exponentials relative to the slice's maximum
  float2 acc[2] = {rows::both(0.f), rows::both(0.f)};
  rows::by_kind(ref, [&](auto far) {
    constexpr bool FAR = decltype(far)::value;
    const float2 c2 = rows::both(c), n2 = rows::both(FAR ? -ref.z : -ref.r);
    rows::for_vectors(s, [&](int v) {
      float2 q[E / 2];
      rows::load_pairs(s, v, q);
#pragma unroll
      for (int i = 0; i < E / 2; ++i)
        acc[i & 1] = rows::add2(acc[i & 1], rows::exp2_pair(rows::log2_pair<FAR>(q[i], c2, n2)));
    });
  });
  acc[0] = rows::add2(acc[0], acc[1]);
  float sum = warp_sum(acc[0].x + acc[0].y);
  if (lane == 0) sh.warp_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = warp_sum(lane < warps ? sh.warp_sums[lane] : 0.f);
    if (lane < parts) {
      Shared* peer = parts > 1 ? cluster.map_shared_rank(&sh, lane) : &sh;
      peer->sum[rank] = sum;
      peer->ref[rank] = ref;
    }
  }
  if (parts > 1)
    cluster.sync();
  else
    __syncthreads();
  // the row's bound, reference and sum: every CTA computes the same
  uint32_t bound = sh.bound[0];
  int best = 0;
  for (int q = 1; q < parts; ++q) {
    bound = min(bound, sh.bound[q]);
    if (sh.sum[q] != 0.f && (sh.sum[best] == 0.f || sh.ref[q].z > sh.ref[best].z)) best = q;
  }
  float total_sum = sh.sum[best];
  for (int q = 0; q < parts; ++q)
    if (q != best && sh.sum[q] != 0.f) total_sum += sh.sum[q] * exp2f(sh.ref[best].log2_of(sh.ref[q], c));

  // Collect: the threads that can hold elements at the bound, then their vectors, a vector per lane.  Without a
  // bound (fewer vectors than r) a short row is taken whole.
  const bool whole = bound <= ordered(-CUDART_INF_F);
  const bool search = total_sum != total_sum || (whole && vocab > kCapacity);  // NaN, or no bound
  Shared* first = parts > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
  unsigned long long* first_list = parts > 1 ? cluster.map_shared_rank(list, 0) : list;
  const auto take = [&](float value, int col) {
    const int to = atomicAdd(&first->taken, 1);
    if (to < kCapacity) first_list[to] = key_of(value, col);
  };
  int found = 0;
  if (!search && whole) {
    for (int i = tid; i < s.nv * E; i += blockDim.x) {
      const int col = s.first + i;
      if (col >= 0 && col < vocab) {
        ++found;
        take(to_f32(s.sm[i]), col);
      }
    }
  } else if (!search) {
    const float least = from_ordered(bound);
    const bool hit = mine >= bound;
    const unsigned who = __ballot_sync(0xffffffffu, hit);
    int at = 0;
    if (lane == 0 && who != 0) at = atomicAdd(&sh.hits, __popc(who));
    at = __shfl_sync(0xffffffffu, at, 0);
    if (hit) sh.hit[at + __popc(who & ((1u << lane) - 1u))] = static_cast<unsigned short>(tid);
    __syncthreads();
    // 16 lanes look through a thread's vectors (it has up to 16 unless a slice is very long)
    const int hits = sh.hits, half = lane & 15;
    for (int h = 2 * warp + (lane >> 4); h < hits; h += 2 * warps) {
      for (int v = sh.hit[h] + half * blockDim.x; v < s.nv; v += 16 * blockDim.x) {
        float2 q[E / 2];
        rows::load_pairs(s, v, q);
        unsigned mask = 0;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          mask |= (q[i].x >= least ? 1u : 0u) << (2 * i);
          mask |= (q[i].y >= least ? 1u : 0u) << (2 * i + 1);
        }
        found += __popc(mask);
        for (; mask != 0; mask &= mask - 1) {
          const int i = v * E + __ffs(mask) - 1;
          take(to_f32(s.sm[i]), s.first + i);
        }
      }
    }
  }
  int total;
  if (parts > 1) {
    found = block_count(found, sh.red);
    if (tid < parts) cluster.map_shared_rank(&sh, tid)->count[0][rank] = found;
    cluster.sync();
    total = 0;
    for (int q = 0; q < parts; ++q) total += sh.count[0][q];
  } else {
    __syncthreads();
    total = sh.taken;
  }

  if (search || total > kCapacity) {
    // the k-th largest key, highest bit first; the column's upper bits are ones in every key
    const int col_bits = 32 - __clz(vocab);
    unsigned long long kth = 0;
    int side = 1;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long trial = kth | (1ull << bit);
      if (bit < 32 && bit >= col_bits) {
        kth = trial;
        continue;
      }
      int n = 0;
      for (int v = tid; v < s.nv; v += blockDim.x) {
        float e[E];
        load_vec<E>(s.sm + v * E, e);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int col = s.first + v * E + i;
          n += col >= 0 && col < vocab && key_of(e[i], col) >= trial;
        }
      }
      n = block_count(n, sh.red);
      if (parts > 1) {
        if (tid < parts) cluster.map_shared_rank(&sh, tid)->count[side][rank] = n;
        cluster.sync();
        n = 0;
        for (int q = 0; q < parts; ++q) n += sh.count[side][q];
        side ^= 1;
      }
      if (n >= k) kth = trial;
    }
    if (rank == 0 && tid == 0) sh.taken = 0;
    if (parts > 1)
      cluster.sync();
    else
      __syncthreads();
    for (int v = tid; v < s.nv; v += blockDim.x) {
      float e[E];
      load_vec<E>(s.sm + v * E, e);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int col = s.first + v * E + i;
        if (col >= 0 && col < vocab && key_of(e[i], col) >= kth) take(e[i], col);
      }
    }
    if (parts > 1)
      cluster.sync();
    else
      __syncthreads();
    total = k;
  }
  if (rank != 0) return;

  // four lanes count the larger keys of each
  for (int i = tid >> 2; i - (lane >> 2) < total; i += blockDim.x / 4) {
    const unsigned long long key = list[min(i, total - 1)];
    int place = 0;
    for (int j = tid & 3; j < total; j += 4) place += list[j] > key;
    place += __shfl_xor_sync(0xffffffffu, place, 1);
    place += __shfl_xor_sync(0xffffffffu, place, 2);
    if ((tid & 3) == 0 && i < total && place < k) {
      values[row * k + place] = from_f32<T>(from_ordered(static_cast<uint32_t>(key >> 32)));
      ids[row * k + place] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
    }
  }
  if (tid == 0) {
    const rows::Ref r = sh.ref[best];
    lse[row] = r.far ? r.z * inv_tau + logf(total_sum) : (r.r + log2f(total_sum)) * CUDART_LN2_F;
  }
}

}  // namespace

void top_logits(const TopLogitsArgs& a, cudaStream_t stream) {
  TTB_CHECK(a.k >= 1 && a.k <= kTopLogitsMaxK && a.k <= a.vocab, "top logits: k must be between 1 and min(256, columns)");
  TTB_CHECK(logits_row_fits(a.vocab, a.type), "top logits: the rows are too long");
  if (a.rows == 0) return;
  if (top_logits_by_ring(a, stream)) return;
  rows::Plan p = rows::plan_rows(a.rows, a.vocab, scalar_bytes(a.type));
  while (p.threads < rows::kMaxThreads && p.threads < 4 * ((a.k + p.parts - 1) / p.parts)) p.threads *= 2;
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
    cfg.numAttrs = p.parts > 1 ? 1 : 0;
    TTB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(a.z), a.ldz, a.vocab, a.k, a.inv_tau,
                                      static_cast<T*>(a.values), a.ids, a.lse, p.per, p.parts, status_ptr()));
  });
}

}  // namespace ttb
