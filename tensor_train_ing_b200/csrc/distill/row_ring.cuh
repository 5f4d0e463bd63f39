// A row of logits in the shared memory of a CTA, or of the CTAs of a cluster, whose warps have roles: `kRingThreads` consumer
// threads work on rows that other warps bring in and finish.
//
// A row is cut into 16-byte vectors counted from the 16-byte boundary at or below its first element, so that
// rows at any element offset are copied in whole aligned vectors; the at most two vectors that reach over the
// row's ends are its edges and are read from global memory element by element.  CTA `rank` of a row has the vectors from
// rank * per on, and its consumer thread t works on the whole ones among the vectors t, t + kRingThreads, ... of them.  They
// arrive in kStages bulk copies with a barrier each, and a stage's memory is given to the CTA's next row as soon as the
// last pass over it is done: a stage is therefore the same vectors of the slice in every row, whatever the row's offset.
#pragma once

#include "row_slice.cuh"

namespace ttb {
namespace rows {

constexpr int kRingWarps = 12;
constexpr int kRingThreads = 32 * kRingWarps;

template <typename T>
struct Span {
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  const T* row;
  int first;   // column of the CTA's vector 0 (negative where that vector starts before the row)
  int lo, hi;  // its whole vectors: [lo, hi)
  int c0, c1;  // its columns: [c0, c1)
  int off;     // elements between the 16-byte boundary and the row's first element
  int stage;   // vectors per stage, a multiple of kRingThreads

  __device__ __forceinline__ Span(const T* r, int cols, int rank, int per) {
    constexpr int E = kVec;
    row = r;
    off = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    const int total = (off + cols + E - 1) / E;
    const int v0 = min(rank * per, total);
    const int nv = min(per, total - v0);
    first = v0 * E - off;
    c0 = min(cols, max(0, first));
    c1 = max(c0, min(cols, first + nv * E));
    lo = first < 0 ? 1 : 0;
    hi = max(lo, first + nv * E > cols ? nv - 1 : nv);
    stage = (per + kStages * kRingThreads - 1) / (kStages * kRingThreads) * kRingThreads;
  }
  __device__ __forceinline__ bool holds(int col) const { return col >= c0 && col < c1; }
  // The stage that brings one of the CTA's columns, or kStages for an edge column.
  __device__ __forceinline__ int stage_of(int col) const {
    const int v = (col - first) / kVec;
    return v >= lo && v < hi ? v / stage : kStages;
  }
  // Edge columns have slots 0..7 (before the first whole vector) and 8..15 (after the last); -1 for no column.
  __device__ __forceinline__ int edge_slot(int col) const {
    const int head = min(c1, first + lo * kVec);
    return col < head ? col - c0 : 8 + col - max(head, first + hi * kVec);
  }
  __device__ __forceinline__ int edge_column(int slot) const {
    const int head = min(c1, first + lo * kVec), tail = max(head, first + hi * kVec);
    const int col = slot < 8 ? c0 + slot : tail + slot - 8;
    return col < (slot < 8 ? head : c1) ? col : -1;
  }
  // One thread: starts the copy of stage g into `sm`.
  __device__ __forceinline__ void load_stage(T* sm, uint64_t* bars, int g) const {
    const int a = max(lo, g * stage), b = min(hi, (g + 1) * stage);
    if (a < b) {
      mbar_arrive_expect_tx(&bars[g], (b - a) * 16);
      bulk_load(sm + a * kVec, row + first + a * kVec, (b - a) * 16, &bars[g]);
    } else {
      mbar_arrive(&bars[g]);
    }
  }
  // f(vector, its number) over the thread's vectors of stage g.  One at a time: the passes are long straight code, and
  // a second copy of them for pairs of vectors costs more in instruction fetches than it gains.
  template <typename F>
  __device__ __forceinline__ void for_stage(const T* sm, int g, F&& f) const {
    const int last = min(hi, (g + 1) * stage);
    int v = g * stage + static_cast<int>(threadIdx.x);
    if (v < lo) v += kRingThreads;
#pragma unroll 1
    for (; v < last; v += kRingThreads) f(*reinterpret_cast<const uint4*>(sm + v * kVec), v);
  }
};

// Whether the barrier's phase completed; false when it, or a wait of another role (`stop`, in shared memory), ran
// out.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_for(uint64_t* bar, int parity, volatile int* stop, uint32_t* status) {
  const auto test = [&] { return CLUSTER ? mbar_test_cluster(bar, parity) : mbar_test(bar, parity); };
  bool ok = test();
  if (!ok) {
    const long long t0 = clock64();
    while (!(ok = test())) {
      if (*stop != 0) break;
      if (clock64() - t0 > kWaitLimitCycles) {
        record_error(status, kErrTimeoutProducer);
        *stop = 1;
        break;
      }
    }
  }
  return ok;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_waits(uint64_t* bar, int parity, volatile int* stop, uint32_t* status) {
  return __all_sync(0xffffffffu, wait_for<CLUSTER>(bar, parity, stop, status));
}
__device__ __forceinline__ void warp_arrives(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// A load that is issued where it stands (the compiler would move a plain one to its use, where its latency shows).
template <typename T>
__device__ __forceinline__ T load_early(const T* p) {
  T v;
  if constexpr (sizeof(T) == 4) {
    uint32_t u;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(u) : "l"(p));
    v = *reinterpret_cast<const T*>(&u);
  } else {
    unsigned short u;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(u) : "l"(p));
    v = *reinterpret_cast<const T*>(&u);
  }
  return v;
}

// The largest of the lanes' values (none NaN), in one instruction.
__device__ __forceinline__ float lanes_max(float v) {
  asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
  return v;
}

// The elements of a vector as pairs.
template <typename T>
__device__ __forceinline__ void to_pairs(const uint4& u, float2 (&p)[Span<T>::kVec / 2]) {
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

// Over vectors (NaN left out): the largest element, the number of a vector that has it, and the largest element of all
// other vectors (or the same, where two vectors share it).
struct Leaders {
  float most, next;
  int where;
  __device__ __forceinline__ Leaders() : most(-__builtin_huge_valf()), next(-__builtin_huge_valf()), where(0) {}
  __device__ __forceinline__ void take(float vector_max, int number) {
    next = fmaxf(next, fminf(vector_max, most));
    if (vector_max > most) where = number;
    most = fmaxf(most, vector_max);
  }
};

// The largest element of a vector (NaN left out).
template <typename T>
__device__ __forceinline__ float max_of(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                       fmaxf(__uint_as_float(u.z), __uint_as_float(u.w))), -CUDART_INF_F);
  } else {
    float a, b;
    unpack2<T>(max2<T>(max2<T>(u.x, u.y), max2<T>(u.z, u.w)), a, b);
    return fmaxf(fmaxf(a, b), -CUDART_INF_F);  // two NaN halves give -inf
  }
}

// A thread's running sums of exp((z - ref) / tau) and, for POW > 0, exp(z - ref), over whatever it has seen.  The
// reference is the largest logit of its first vector that has one.  While `see` is called before every vector it moves when
// one exceeds it by more than 2^40, at the temperature or at 1, so that no element adds more to either sum.  Vectors added
// without have no maximum to take, which is a fifth of the work and a branch that keeps the next one's loads and
// exponentials from starting, but their sums may grow past kSafeSum: then `overflowed`, and the sums have to be taken again.
//
// kSafeSum lies far below the largest fp32 number because of what is made of the sums.  The sums of 384 threads and 8 CTAs
// add up to less than 2^72; 1 / sum, times a loss scale and a weight, stays a normal number and its quotient in the range
// of the fast division (denominators up to 2^126); and a sum that another's larger reference scales by less
// than 2^-126, that is to zero, is below 2^-54 of that other's.
constexpr float kSafeSum = 1.152921504606846976e18f;  // 2^60
template <int POW>
struct Sums {
  Ref ref, ref1;
  bool set;  // whether any finite logit has been seen; until then the reference is 0
  float2 acc[2], acc1[2];

  __device__ __forceinline__ explicit Sums(float c) : ref(0.f, c), ref1(0.f, c), set(false) {
    acc[0] = acc[1] = acc1[0] = acc1[1] = both(0.f);
  }
  // to this logit, `above` the reference by so many powers of two
  __device__ __forceinline__ void move(float logit, float above, float c) {
    const Ref next(logit, c), next1 = ref_at_one<POW>(next);
    if (set && !overflowed()) {  // sums past kSafeSum stay so: a factor that underflows would hide what they lose
      const float step = next.excess(c) - above;
      const float2 f = both(fast_exp2(step));
      acc[0] = mul2(acc[0], f);
      acc[1] = mul2(acc[1], f);
      if (POW != 0) {
        const float2 f1 = both(fast_exp2(log2_at_one<POW>(step, next1, ref1)));
        acc1[0] = mul2(acc1[0], f1);
        acc1[1] = mul2(acc1[1], f1);
      }
    }
    ref = next;
    ref1 = next1;
    set = true;
  }
  // 40, as an exponent at the temperature: an exponential at 1 has tau times the exponent (tau = log2(e) / c).
  __device__ __forceinline__ static float most_above(float c) {
    if (POW == 0) return 40.f;
    return POW == 1 ? 40.f * fminf(1.f, c * CUDART_LN2_F) : 40.f / POW;
  }
  // before adding logits of which `top` is the largest
  __device__ __forceinline__ void see(float top, float c) {
    const float above = ref.log2_of(top, c);
    if ((!set || above > most_above(c)) && fabsf(top) < CUDART_INF_F) move(top, above, c);
  }
  // Whether vectors may be added without `see` from here on: all of the warp's threads have ordinary references.  One far
  // below the warp's largest (a thread whose first vectors are masked) moves there, so that it will not overflow.
  __device__ __forceinline__ bool settle(float c) {
    see(lanes_max(set ? ref.z : -CUDART_INF_F), c);
    return __all_sync(0xffffffffu, set && !ref.far);
  }
  template <bool FAR>
  __device__ __forceinline__ void add(float2 z, int i, float c) {
    const float2 e = exp2_pair(log2_pair<FAR>(z, both(c), both(FAR ? -ref.z : -ref.r)));
    acc[i & 1] = add2(acc[i & 1], e);
    if constexpr (POW == 2) acc1[i & 1] = fma2(e, e, acc1[i & 1]);
    if constexpr (POW == 1 || POW == 4) acc1[i & 1] = add2(acc1[i & 1], at_one<POW, FAR>(e, z, ref1));
  }
  template <typename T, bool FAR>
  __device__ __forceinline__ void add_vector(const uint4& u, float c) {
    float2 q[Span<T>::kVec / 2];
    to_pairs<T>(u, q);
#pragma unroll
    for (int i = 0; i < Span<T>::kVec / 2; ++i) add<FAR>(q[i], i, c);
  }
  template <typename T>
  __device__ __forceinline__ void add_seen(const uint4& u, float c) {
    if (ref.far)
      add_vector<T, true>(u, c);
    else
      add_vector<T, false>(u, c);
  }
  __device__ __forceinline__ void add_one(float z, float c) {
    see(z, c);
    const float2 pair = make_float2(z, -CUDART_INF_F);
    if (ref.far)
      add<true>(pair, 0, c);
    else
      add<false>(pair, 0, c);
  }
  __device__ __forceinline__ bool overflowed() const { return !(sum() < kSafeSum) || !(sum1() < kSafeSum); }
  __device__ __forceinline__ float sum() const { return (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y); }
  __device__ __forceinline__ float sum1() const { return (acc1[0].x + acc1[0].y) + (acc1[1].x + acc1[1].y); }
};

// sum 2^log2; nothing, and infinity, stay what they are.
__device__ __forceinline__ float rescaled(float sum, float log2) {
  return sum != 0.f && sum < CUDART_INF_F ? sum * fast_exp2(log2) : sum;
}

// What a warp's threads have summed, relative to one reference (lane 0 has the sums).
struct WarpSum {
  float z;  // the reference logit; -inf where the warp has seen no finite logit
  float sum, sum1;
};
template <int POW>
__device__ __forceinline__ WarpSum warp_total(const Sums<POW>& s, float c) {
  WarpSum w;
  w.z = lanes_max(s.set ? s.ref.z : -CUDART_INF_F);
  const Ref ref(w.z == -CUDART_INF_F ? 0.f : w.z, c);
  w.sum = s.sum();
  const float step = ref.log2_of(s.ref, c);
  w.sum = rescaled(w.sum, step);
  w.sum = warp_sum(w.sum);
  w.sum1 = 0.f;
  if (POW != 0) {
    w.sum1 = s.sum1();
    w.sum1 = rescaled(w.sum1, log2_at_one<POW>(step, ref_at_one<POW>(ref), s.ref1));
    w.sum1 = warp_sum(w.sum1);
  }
  return w;
}

}  // namespace rows
}  // namespace ttb
