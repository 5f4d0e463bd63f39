// What the two kernels of the distillation loss share (formulas in distill_api.h).
#pragma once

#include "distill_api.h"
#include "row_slice.cuh"

namespace ttb {
namespace distill {

struct Params {
  long long rows;
  int vocab, k, per, parts, dz_cols;
  bool ids64;
  float inv_tau, tau, kd, ce;
  const void* ids;
  const void* t;
  ScalarType t_type;
  const float* teacher_lse;
  const long long* targets;
  const float* scale;
  const float* factor;
  int factor_step;
  float* loss;
  long long ldz, lddz;
  uint32_t* status;
};

__device__ __forceinline__ float teacher_logit(const Params& p, long long i) {
  if (p.t_type == ScalarType::kF32) return static_cast<const float*>(p.t)[i];
  if (p.t_type == ScalarType::kBF16) return to_f32(static_cast<const __nv_bfloat16*>(p.t)[i]);
  return to_f32(static_cast<const __half*>(p.t)[i]);
}

// What a kernel forms: the loss, its gradient too, or the gradient once more with a factor (DistillArgs::factor; kernels of
// their own, so that the others carry no code for it).
constexpr int kLoss = 0, kGradient = 1, kAgain = 2;

template <int FORM>
__device__ __forceinline__ bool nothing_to_do(const Params& p) {
  return FORM == kAgain && p.factor_step == 0 && *p.factor == 1.f;
}
// What multiplies a row's loss and gradient, `scale` being what multiplies all rows'.
__device__ __forceinline__ float scale_of_all(const Params& p) { return p.scale != nullptr ? *p.scale : 1.f; }
template <int FORM>
__device__ __forceinline__ float scale_of(const Params& p, float scale, long long row) {
  return FORM == kAgain ? scale * p.factor[row * p.factor_step] : scale;
}

// The smem element a listed column's slot holds while entries compete for it, as bits of a finite value.
template <typename T>
__device__ __forceinline__ void put_mark(T* p, int i) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<int*>(p) = i;
  else *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(i);
}
template <typename T>
__device__ __forceinline__ int get_mark(const T* p) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const int*>(p);
  else return *reinterpret_cast<const unsigned short*>(p);
}

// Whether no entry before i names entry i's column.  Which of several entries stands for a column decides where its exponential
// is added; the competition for its slot has some winner, this one has the same in every run.
template <typename E>
__device__ __noinline__ bool first_of_column(const E* list, int i) {
  for (int j = 0; j < i; ++j)
    if (list[j].col == list[i].col) return false;
  return true;
}

// Threads first, first + step, ... write the row's zeros: 16 bytes each between the ragged ends.
template <typename T>
__device__ __forceinline__ void zero_row(T* row, int cols, int first, int step) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const int head = min(cols, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / sizeof(T)));
  const int vecs = (cols - head) / E;
  for (int i = first; i < head; i += step) row[i] = from_f32<T>(0.f);
  for (int i = first; i < vecs; i += step) reinterpret_cast<uint4*>(row + head)[i] = make_uint4(0, 0, 0, 0);
  for (int i = head + vecs * E + first; i < cols; i += step) row[i] = from_f32<T>(0.f);
}

// f(logits, gradient) with the pointers' types; f(std::integral_constant<int, POW>).
template <typename F>
void with_kernel_types(const DistillArgs& a, F&& f) {
  with_type(a.z_type, [&](auto* tz) {
    using TZ = std::remove_pointer_t<decltype(tz)>;
    if (a.dz != nullptr && a.dz_type != a.z_type)
      f(static_cast<const TZ*>(a.z), static_cast<__nv_bfloat16*>(a.dz));
    else
      f(static_cast<const TZ*>(a.z), static_cast<TZ*>(a.dz));
  });
}
template <typename F>
void with_pow(int pow, F&& f) {
  switch (pow) {
    case 0: return f(std::integral_constant<int, 0>{});
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 4>{});
  }
}

// f(std::integral_constant<int, FORM>) for these types.
template <typename TZ, typename TG, typename F>
void with_form(const DistillArgs& a, F&& f) {
  if (a.dz == nullptr) return f(std::integral_constant<int, kLoss>{});
  if (a.factor == nullptr) return f(std::integral_constant<int, kGradient>{});
  if constexpr (std::is_same_v<TZ, __half> && std::is_same_v<TG, __half>)
    f(std::integral_constant<int, kAgain>{});
}

// The kernel for many long rows (distill_ring.cu); false where it does not apply.
bool loss_by_ring(const DistillArgs& a, const Params& p, int pow, cudaStream_t stream);

}  // namespace distill
}  // namespace ttb
