// What the two kernels of the top logits share.
#pragma once

#include "distill_api.h"
#include "row_slice.cuh"

namespace ttb {
namespace top {

constexpr int kCapacity = 640;  // collected elements: about 1.7 times the largest k

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

// A value that at least r and, where the values allow it, few more than r of `count` maxima reach (0 where
// fewer than r have elements); FOLD of them count as one.  One warp; the common leading bits are skipped.
template <typename T, int FOLD = 1>
__device__ __forceinline__ uint32_t find_bound(const uint32_t* maxima, int count, int r) {
  constexpr int kMost = 16;
  const int lane = threadIdx.x & 31, each = count / 32 / FOLD;
  uint32_t m[kMost];
  uint32_t all = 0xFFFFFFFFu, any = 0u;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    m[i] = i < each ? maxima[i * FOLD * 32 + lane] : 0u;
#pragma unroll
    for (int f = 1; f < FOLD; ++f)
      if (i < each) m[i] = max(m[i], maxima[(i * FOLD + f) * 32 + lane]);
    if (i < each) {
      all &= m[i];
      any |= m[i];
    }
  }
  all = __reduce_and_sync(0xffffffffu, all);
  any = __reduce_or_sync(0xffffffffu, any);
  const uint32_t differ = all ^ any;
  if (r > 32 * each) return 0u;
  if (differ == 0) return all;
  const int top = 31 - __clz(differ);
  uint32_t bound = top == 31 ? 0u : all & ~((2u << top) - 1u);
  for (int bit = top; bit >= lowest_bit<T>(); --bit) {
    const uint32_t trial = bound | (1u << bit);
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) c += m[i] >= trial;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= r) bound = trial;
    if (c >= r && c <= r + r / 8) break;  // close enough: a higher bound would only shorten the list a little
  }
  return bound;
}

// The same over maxima left in shared memory, one for one: slower, and closer where r is no small part of the count.
template <typename T>
__device__ __noinline__ uint32_t find_close_bound(const uint32_t* maxima, int count, int r) {
  const int lane = threadIdx.x & 31;
  uint32_t bound = 0;
  for (int bit = 31; bit >= lowest_bit<T>(); --bit) {
    const uint32_t trial = bound | (1u << bit);
    int c = 0;
#pragma unroll 8
    for (int i = lane; i < count; i += 32) c += maxima[i] >= trial;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= r) bound = trial;
    if (c >= r && c <= r + r / 16) break;
  }
  return bound;
}

// The kernel for many long rows (top_ring.cu); false where it does not apply.
bool top_logits_by_ring(const TopLogitsArgs& a, cudaStream_t stream);

}  // namespace top
}  // namespace ttb
