// A row of logits held in the shared memory of a cluster: CTA `rank` of the row's `parts` CTAs keeps the
// `per` 16-byte vectors from rank * per on.  Vectors are counted from the 16-byte boundary at or below
// the row's first element, so that rows at any element offset are copied in aligned 16-byte pieces;
// positions outside the row (before its first element, past its last) hold -inf.
#pragma once

#include <cooperative_groups.h>
#include <math_constants.h>

#include "../common/sm100.cuh"
#include "../common/vec.cuh"

namespace ttb {
namespace rows {

namespace cg = cooperative_groups;

template <typename T>
struct Slice {
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  T* sm;      // element i of the slice is row element first + i
  int first;  // negative in slice 0 of a row that starts off a 16-byte boundary
  int nv;     // vectors in this slice
  int off;    // elements between the 16-byte boundary and the row's first element

  __device__ __forceinline__ int begin(int cols) const { return max(0, -first); }
  __device__ __forceinline__ bool holds(int col) const { return col >= first && col < first + nv * kVec; }
};

template <typename T>
__device__ __forceinline__ T neg_inf() {
  return from_f32<T>(-CUDART_INF_F);
}

// Issues the asynchronous copies of this CTA's slice; finish_load waits for them.
template <typename T>
__device__ __forceinline__ Slice<T> start_load(T* sm, const T* row, int cols, int rank, int per) {
  constexpr int E = Slice<T>::kVec;
  Slice<T> s;
  s.sm = sm;
  s.off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int total = (s.off + cols + E - 1) / E;
  const int v0 = min(rank * per, total);
  s.nv = min(per, total - v0);
  s.first = v0 * E - s.off;
  for (int v = threadIdx.x; v < s.nv; v += blockDim.x) {
    const int col = s.first + v * E;
    if (col >= 0 && col + E <= cols) {
      cp_async16(smem_u32(sm + v * E), row + col);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) sm[v * E + i] = (col + i >= 0 && col + i < cols) ? row[col + i] : neg_inf<T>();
    }
  }
  cp_async_commit();
  return s;
}
__device__ __forceinline__ void finish_load() {
  cp_async_wait<0>();
  __syncthreads();
}

__device__ __forceinline__ float fast_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// How rows are spread: `parts` CTAs per row (a cluster), `per` vectors each, `threads` threads each.
struct Plan {
  int parts, per, threads;
  size_t slice_bytes;
};

constexpr int kMaxParts = 8;                  // the portable cluster size
constexpr size_t kMaxSliceBytes = 192 * 1024;  // of the 227 KB a CTA may hold; the rest is for lists

Plan plan_rows(long long rows, int cols, int elem_bytes);

}  // namespace rows
}  // namespace ttb
