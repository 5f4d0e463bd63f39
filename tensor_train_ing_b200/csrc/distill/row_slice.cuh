// A row of logits held in the shared memory of a cluster: CTA `rank` of the row's `parts` CTAs keeps the
// `per` 16-byte vectors from rank * per on.  Vectors are counted from the 16-byte boundary at or below
// the row's first element, so that rows at any element offset are copied in aligned 16-byte pieces;
// positions outside the row (before its first element, past its last) hold -inf.
//
// Thread t copies, and in every later pass works on, the vectors t, t + threads, ... of its slice: a pass
// over the slice needs no block barrier after the copies, only the thread's own copies to have arrived.
#pragma once

#include <cooperative_groups.h>
#include <math_constants.h>

#include "../common/sm100.cuh"
#include "../common/vec.cuh"

namespace ttb {
namespace rows {

namespace cg = cooperative_groups;

constexpr int kStages = 4;  // groups of copies that can be waited for one after the other

template <typename T>
struct Slice {
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  T* sm;       // element i of the slice is row element first + i
  int first;   // negative in slice 0 of a row that starts off a 16-byte boundary
  int nv;      // vectors in this slice
  int off;     // elements between the 16-byte boundary and the row's first element
  int stage;   // vectors per stage and thread

  __device__ __forceinline__ bool holds(int col) const { return col >= first && col < first + nv * kVec; }
};

template <typename T>
__device__ __forceinline__ T neg_inf() {
  return from_f32<T>(-CUDART_INF_F);
}

// Issues the asynchronous copies of this CTA's slice in kStages groups.
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
  const int each = (s.nv + blockDim.x - 1) / blockDim.x;
  s.stage = (each + kStages - 1) / kStages;
  int v = threadIdx.x;
#pragma unroll
  for (int g = 0; g < kStages; ++g) {
    for (int i = 0; i < s.stage && v < s.nv; ++i, v += blockDim.x) {
      const int col = s.first + v * E;
      if (col >= 0 && col + E <= cols) {
        cp_async16(smem_u32(sm + v * E), row + col);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) sm[v * E + e] = (col + e >= 0 && col + e < cols) ? row[col + e] : neg_inf<T>();
      }
    }
    cp_async_commit();
  }
  return s;
}

// The largest element of the thread's vectors (NaN left out), taken as the copies arrive; all of
// the thread's own copies have arrived when it returns.
template <typename T>
__device__ __forceinline__ float max_while_loading(const Slice<T>& s) {
  constexpr int E = Slice<T>::kVec;
  float mx = -CUDART_INF_F;
  uint32_t packed = 0;  // two running maxima of a 16-bit type
  if constexpr (sizeof(T) == 2) packed = pack2<T>(mx, mx);
  int v = threadIdx.x;
#pragma unroll
  for (int g = 0; g < kStages; ++g) {
    if (g == 0) cp_async_wait<3>();
    if (g == 1) cp_async_wait<2>();
    if (g == 2) cp_async_wait<1>();
    if (g == 3) cp_async_wait<0>();
    for (int i = 0; i < s.stage && v < s.nv; ++i, v += blockDim.x) {
      const uint4 u = *reinterpret_cast<const uint4*>(s.sm + v * E);
      if constexpr (sizeof(T) == 4) {
        mx = fmaxf(fmaxf(mx, fmaxf(__uint_as_float(u.x), __uint_as_float(u.y))),
                   fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
      } else {
        packed = max2<T>(max2<T>(packed, max2<T>(u.x, u.y)), max2<T>(u.z, u.w));
      }
    }
  }
  if constexpr (sizeof(T) == 2) {
    float lo, hi;
    unpack2<T>(packed, lo, hi);
    mx = fmaxf(lo, hi);
  }
  return mx;
}

__device__ __forceinline__ float fast_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Pairs of fp32 numbers for the packed fp32 instructions (one instruction, two elements).
__device__ __forceinline__ unsigned long long bits(float2 a) { return *reinterpret_cast<unsigned long long*>(&a); }
__device__ __forceinline__ float2 pair(unsigned long long a) { return *reinterpret_cast<float2*>(&a); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return pair(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Vector v of the slice as pairs.
template <typename T>
__device__ __forceinline__ void load_pairs(const Slice<T>& s, int v, float2 (&p)[Slice<T>::kVec / 2]) {
  const uint4 u = *reinterpret_cast<const uint4*>(s.sm + v * Slice<T>::kVec);
  if constexpr (sizeof(T) == 4) {
    p[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    p[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    unpack2<T>(u.x, p[0].x, p[0].y);
    unpack2<T>(u.y, p[1].x, p[1].y);
    unpack2<T>(u.z, p[2].x, p[2].y);
    unpack2<T>(u.w, p[3].x, p[3].y);
  }
}

// How rows are spread: `parts` CTAs per row (a cluster), `per` vectors each, `threads` threads each.
struct Plan {
  int parts, per, threads;
  size_t slice_bytes;
};

constexpr int kMaxParts = 8;                   // the portable cluster size
constexpr int kMaxThreads = 512;
constexpr size_t kMaxSliceBytes = 192 * 1024;  // of the 227 KB a CTA may hold; the rest is for lists

Plan plan_rows(long long rows, int cols, int elem_bytes);

}  // namespace rows
}  // namespace ttb
