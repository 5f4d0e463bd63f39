// Row operators on logits for distillation: a teacher's top logits and the loss against them.
//
//   top logits   per row the k largest logits in descending order (equal logits: the lower column first; NaN counts
//                as the largest value), their columns, and log sum_j exp(z_j / tau)
//
//   loss         a_i = t_i / tau over the teacher's listed columns c_i (entries with c_i < 0 are absent)
//                p_i = exp(a_i - L): L is the teacher's log-sum-exp over all its columns where given (then
//                m = 1 - sum_i p_i is its mass on all other columns), else that of the listed a_i (m = 0)
//                q = softmax(z / tau), q_rest = sum of q_j over the columns that are not listed
//                KL = sum_i p_i (log p_i - log q_{c_i}) + m (log m - log q_rest)
//                loss = scale (kd tau^2 KL + ce (log sum_j exp z_j - z_target))
//   gradient     dz_j = scale (kd tau (q_j (P + m) - p_j) + ce (softmax(z)_j - [j = target]))      for listed j
//                dz_j = scale (kd tau q_j (P + m - m / q_rest) + ce (softmax(z)_j - [j = target])) for the others
//                with P = sum_i p_i
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/dtype.h"

namespace ttb {

constexpr int kTopLogitsMaxK = 256;
constexpr int kDistillMaxList = 1024;
// Mass outside the teacher's list at or below this counts as none: L is a number around 10 held in fp32, so
// 1 - sum p is uncertain by about 2^-20, and log of a rounding error is no information.
constexpr float kDistillLeastRest = 9.5367431640625e-07f;

// Whether rows of `cols` elements of this type fit the kernels (a row is held in the shared memory of one cluster).
bool logits_row_fits(int cols, ScalarType type);

struct TopLogitsArgs {
  const void* z;  // [rows, vocab], rows ldz elements apart
  long long ldz;
  ScalarType type;
  long long rows;
  int vocab, k;
  float inv_tau;
  void* values;  // [rows, k] of z's type
  int* ids;      // [rows, k]
  float* lse;    // [rows]
};
void top_logits(const TopLogitsArgs& a, cudaStream_t stream);

struct DistillArgs {
  const void* z;  // [rows, vocab], rows ldz elements apart
  long long ldz;
  ScalarType z_type;
  long long rows;
  int vocab;
  const void* ids;  // [rows, k] int32 or int64, dense
  bool ids64;
  const void* t;  // [rows, k], dense
  ScalarType t_type;
  int k;
  const float* teacher_lse;   // [rows] or null
  const long long* targets;   // [rows] or null; a negative target leaves its row out
  float tau, kd, ce;
  const float* scale;  // device scalar or null (1)
  // With an fp16 gradient of fp16 logits: what multiplies row r besides, factor[r * factor_step], or null (1).  A single factor
  // (step 0) of 1 leaves dz as it is: it holds the answer already.  The loss is not written then.
  const float* factor;
  int factor_step;
  float* loss;         // [rows]; with a factor unused
  void* dz;            // null: no gradient.  [rows, dz_cols], rows lddz apart; columns past vocab are written as zeros
  long long lddz;
  int dz_cols;
  ScalarType dz_type;  // z's type, or bf16 with z fp32
  uint32_t* status;
};
void distill_loss(const DistillArgs& a, cudaStream_t stream);

// Row r of dz times g[r * gstep] (gstep 0: one factor for all rows), rounded to dz's type; rows whose factor is 1
// are not touched.
void scale_in_place(void* dz, ScalarType type, long long rows, int cols, long long ld, const float* g, int gstep,
                    cudaStream_t stream);

}  // namespace ttb
