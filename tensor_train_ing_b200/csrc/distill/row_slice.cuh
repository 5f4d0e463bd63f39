// A row of logits held in the shared memory of a cluster: CTA `rank` of the row's `parts` CTAs keeps the
// `per` 16-byte vectors from rank * per on.  Vectors are counted from the 16-byte boundary at or below
// the row's first element, so that rows at any element offset are copied in aligned 16-byte pieces;
// positions outside the row (before its first element, past its last) hold -inf.
//
// The slice arrives in kStages bulk copies with a barrier each.  Thread t works, in every pass, on the vectors t, t +
// threads, ... of the slice, and stage g holds a whole number of such rounds.
#pragma once

#include <cooperative_groups.h>
#include <math_constants.h>

#include "../common/sm100.cuh"
#include "../common/vec.cuh"

namespace ttb {
namespace rows {

namespace cg = cooperative_groups;

constexpr int kStages = 4;

template <typename T>
struct Slice {
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  T* sm;       // element i of the slice is row element first + i
  int first;   // negative in slice 0 of a row that starts off a 16-byte boundary
  int nv;      // vectors in this slice
  int off;     // elements between the 16-byte boundary and the row's first element
  int rounds;  // vectors that every thread has; the threads below nv - rounds * threads have one more
  int stage;   // rounds per stage

  __device__ __forceinline__ bool holds(int col) const { return col >= first && col < first + nv * kVec; }
};

// f(v) for each of the thread's vectors.
template <typename T, typename F>
__device__ __forceinline__ void for_vectors(const Slice<T>& s, F&& f) {
  int v = threadIdx.x;
#pragma unroll 2
  for (int i = 0; i < s.rounds; ++i, v += blockDim.x) f(v);
  if (v < s.nv) f(v);
}

template <typename T>
__device__ __forceinline__ T neg_inf() {
  return from_f32<T>(-CUDART_INF_F);
}

// Starts the copies of this CTA's slice (all threads; ends with a block barrier).  The at most two vectors that reach
// over the row's ends are read element by element by the threads that own them.
template <typename T>
__device__ __forceinline__ Slice<T> start_load(T* sm, uint64_t (&bars)[kStages], const T* row, int cols, int rank,
                                               int per) {
  constexpr int E = Slice<T>::kVec;
  Slice<T> s;
  s.sm = sm;
  s.off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int total = (s.off + cols + E - 1) / E;
  const int v0 = min(rank * per, total);
  s.nv = min(per, total - v0);
  s.first = v0 * E - s.off;
  s.rounds = s.nv / static_cast<int>(blockDim.x);
  s.stage = s.rounds / kStages + 1;
  const int lo = s.first < 0 ? 1 : 0;                                // whole vectors: [lo, hi)
  const int hi = s.first + s.nv * E > cols ? s.nv - 1 : s.nv;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int g = 0; g < kStages; ++g) mbar_init(&bars[g], 1);
    fence_mbar_init();
#pragma unroll
    for (int g = 0; g < kStages; ++g) {
      const int a = max(lo, g * s.stage * static_cast<int>(blockDim.x));
      const int b = min(hi, (g + 1) * s.stage * static_cast<int>(blockDim.x));
      if (a < b) {
        mbar_arrive_expect_tx(&bars[g], (b - a) * 16);
        bulk_load(sm + a * E, row + s.first + a * E, (b - a) * 16, &bars[g]);
      } else {
        mbar_arrive(&bars[g]);
      }
    }
  }
  const int edges[2] = {lo == 1 ? 0 : -1, hi < s.nv && !(lo == 1 && s.nv == 1) ? s.nv - 1 : -1};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int v = edges[q];
    if (v >= 0 && v % static_cast<int>(blockDim.x) == threadIdx.x) {
      const int col = s.first + v * E;
#pragma unroll
      for (int e = 0; e < E; ++e) sm[v * E + e] = (col + e >= 0 && col + e < cols) ? row[col + e] : neg_inf<T>();
    }
  }
  __syncthreads();
  return s;
}

// Waits for stage g.  The wait is bounded; one that runs out is reported and waited for once more, so that the
// copy does not outlive the CTA.
__device__ __forceinline__ void wait_stage(uint64_t* bar, uint32_t* status) {
  if (!mbar_wait(bar, 0, status, kErrTimeoutProducer)) mbar_wait(bar, 0, status, kErrTimeoutProducer);
}

// The largest element of the thread's vectors (NaN left out), taken as the stages arrive; the whole slice has
// arrived when it returns.
template <typename T>
__device__ __forceinline__ float max_while_loading(const Slice<T>& s, uint64_t (&bars)[kStages], uint32_t* status) {
  constexpr int E = Slice<T>::kVec;
  float mx = -CUDART_INF_F;
  uint32_t packed = 0;  // two running maxima of a 16-bit type
  if constexpr (sizeof(T) == 2) packed = pack2<T>(mx, mx);
  auto take = [&](int v) {
    const uint4 u = *reinterpret_cast<const uint4*>(s.sm + v * E);
    if constexpr (sizeof(T) == 4)
      mx = fmaxf(fmaxf(mx, fmaxf(__uint_as_float(u.x), __uint_as_float(u.y))),
                 fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    else
      packed = max2<T>(max2<T>(packed, max2<T>(u.x, u.y)), max2<T>(u.z, u.w));
  };
  int v = threadIdx.x, done = 0;
#pragma unroll
  for (int g = 0; g < kStages; ++g) {
    wait_stage(&bars[g], status);
    const int end = min(s.rounds, (g + 1) * s.stage);
#pragma unroll 2
    for (; done < end; ++done, v += blockDim.x) take(v);
  }
  if (v < s.nv) take(v);
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

// Exponentials are taken as powers of two of z c - r, c = log2(e) / tau, in one fused multiply-add: r is the fp32
// number nearest to (largest logit) c, and everything about a row is kept relative to 2^r, so r's rounding
// cancels.  That takes an r whose rounding is small itself: at a product of 2^24 it is up to 1/2, and at 2^34 (a row
// masked with -1e10) it would be an exponent of 512.  From 2^24 on, at the temperature or at 1, z is instead compared with the logit
// itself first, and everything is relative to exp(logit / tau).
struct Ref {
  float z, r;  // the reference logit and z c
  bool far;    // compared by logits
  __device__ __forceinline__ Ref() {}
  __device__ __forceinline__ Ref(float zmax, float c) {
    z = isfinite(zmax) ? zmax : 0.f;
    far = !(fabsf(z) * fmaxf(c, CUDART_L2E_F) < 16777216.f);
    r = z * c;
  }
  // log2 of exp((v - reference) / tau)
  __device__ __forceinline__ float log2_of(float v, float c) const { return far ? (v - z) * c : fmaf(v, c, -r); }
  // log2 of exp(logit / tau) over what the reference stands for, exactly
  __device__ __forceinline__ float excess(float c) const { return far ? 0.f : fmaf(z, c, -r); }
  // log2 of another reference, of the same row, over this one, whatever their kinds
  __device__ __forceinline__ float log2_of(const Ref& o, float c) const { return excess(c) - o.log2_of(z, c); }
  // the natural logarithm of the same (c times the type's lowest value is no fp32 number)
  __device__ __forceinline__ float log_of(const Ref& o, float c, float inv_tau) const {
    return fmaf(o.z - z, inv_tau, (excess(c) - o.excess(c)) * CUDART_LN2_F);
  }
};

// The exponents of a pair; FAR: ref.far, n = -ref.z there, else -ref.r.
template <bool FAR>
__device__ __forceinline__ float2 log2_pair(float2 q, float2 c, float2 n) {
  return FAR ? mul2(add2(q, n), c) : fma2(q, c, n);
}
__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }

// The reference at temperature 1 that goes with `ref` at tau: with e^POW for the exponentials, exactly POW times it.
template <int POW>
__device__ __forceinline__ Ref ref_at_one(const Ref& ref) {
  Ref r = ref;
  if constexpr (POW == 1) r.r = ref.z * CUDART_L2E_F;
  if constexpr (POW > 1) r.r = POW * ref.r;
  return r;
}
// log2 of o1 over ref1, references at temperature 1, where `step` is that of the references at tau that they go with.
template <int POW>
__device__ __forceinline__ float log2_at_one(float step, const Ref& ref1, const Ref& o1) {
  return POW == 1 ? ref1.log2_of(o1, CUDART_L2E_F) : POW * step;
}

// exp(z - reference) of a pair of logits, from e = exp((z - reference) / tau) where POW says so.
template <int POW, bool FAR>
__device__ __forceinline__ float2 at_one(float2 e, float2 z, const Ref& ref1) {
  if constexpr (POW == 2) {
    return mul2(e, e);
  } else if constexpr (POW == 4) {
    const float2 sq = mul2(e, e);
    return mul2(sq, sq);
  } else {
    return exp2_pair(
        log2_pair<FAR>(z, both(CUDART_L2E_F), both(FAR ? -ref1.z : -ref1.r)));
  }
}

// f(std::bool_constant<ref.far>): the passes are compiled for both kinds of row.
template <typename F>
__device__ __forceinline__ void by_kind(const Ref& ref, F&& f) {
  if (ref.far)
    f(std::true_type{});
  else
    f(std::false_type{});
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
