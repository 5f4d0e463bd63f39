// Distillation from a teacher's top logits: the loss of every row and, in the same pass over the logits, its
// gradient (formulas in distill_api.h).
//
// A row sits in the shared memory of a cluster, usually of one CTA (row_slice.cuh), so the gradient needs no second
// read of it.  While it arrives, every thread takes the maximum of its elements and the first warp reads the
// teacher's list with the student's logits at it.  The listed columns are then taken out of the slice
// (replaced by -inf): what the passes over the slice sum is the rest of the row, whose mass q_rest is thereby never the
// difference of two nearly equal numbers.  With R the row's reference (its largest logit), every unlisted
// column's gradient is
//     exp((z_j - R) / tau) A + exp(z_j - R) B,
//     A = scale kd tau ((P + m) / T - m / S),  S, T = sums of exp((z - R) / tau) over the rest and the row
//     B = scale ce / T1,                       T1 = sum of exp(z - R) over the row
// and the few listed columns and the target are written after the others.  Where the rest lies so far below the list that S or
// much of it vanishes in fp32, it is summed again relative to the rest's own largest logit.
//
// POW: how exp(z - R) of the cross-entropy follows from e = exp((z - R) / tau) of the divergence: not needed or the
// same (0), e^2 or e^4 for the temperatures 2 and 4 (a product is cheaper than a second exponential: the
// special-function unit gives 16 a cycle and SM, and two more per element would bound 16-bit logits), else (1) by
// another exponential.
//
// Few rows, and rows shorter than the persistent kernel's.  Bound by what a row waits for: its copy, the list, and the three
// barriers between maximum, sums and gradient, filled only by the SM's other CTAs.  8288 rows of 16384 bf16 logits, 64 listed:
// 95 us for the loss (42 us for the bytes), 136 us with the gradient (83 us).  Six CTAs of 256 threads share an SM there, so
// the registers are held to 40: 57 leave four of them and cost a quarter of the time.
#include "../common/host.h"
#include "distill_common.cuh"

namespace ttb {
namespace {

using distill::first_of_column;
using distill::get_mark;
using distill::Params;
using distill::put_mark;
using distill::teacher_logit;
using distill::zero_row;

using rows::Slice;
namespace cg = cooperative_groups;

// Below this the rest's sum is taken again relative to its own largest logit.  Exponentials vanish below 2^-126; of a sum
// of 2^-64 and more what vanished is less than 2^-62 an element, less than 2^-42 in all.
constexpr float kLeastRestSum = 5.421010862427522e-20f;  // 2^-64

struct Part {  // what one CTA knows of its slice; sums are relative to its references at tau and at 1
  rows::Ref ref, ref1;
  float rest, rest1;  // unlisted columns, at tau and at 1
  float list, list1;  // listed columns (each counted once)
  int listed;
};

struct Shared {
  uint64_t bars[rows::kStages];
  Part part[rows::kMaxParts], again_part[rows::kMaxParts];
  float red[rows::kMaxThreads / 32][4];
  float red_max[rows::kMaxThreads / 32];
  float target_logit;
  float mass, rest;  // P and m
  float scale;
  // the row's scalars for the gradient: q_j = 2^(z_j c - top) inv_sum; the passes over the slice use ref
  rows::Ref ref, ref1, top, top1;
  float A, B, inv_sum, inv_sum1, all_mass;
  int again, repeats, target_listed, listed;
};

// Entry i of the shared-memory copy of the teacher's list.
struct Entry {
  int col;      // -1: absent
  float logp, p;  // log p_i and p_i (0: no mass)
  float z;      // the student's logit at col
  int owner;    // whether this entry stands for its column here (the first CTA-local entry with this column)
};

template <typename TZ, typename TG, int FORM, int POW>
__global__ void __launch_bounds__(rows::kMaxThreads, 3) distill_kernel(const TZ* __restrict__ z, TG* __restrict__ dz,
                                                                      const __grid_constant__ Params p) {
  constexpr int E = Slice<TZ>::kVec;
  constexpr bool GRAD = FORM != distill::kLoss;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  if (distill::nothing_to_do<FORM>(p)) return;  // the same for the whole grid
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = p.parts, rank = parts > 1 ? cluster.block_rank() : 0;
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  auto* list = reinterpret_cast<Entry*>(smem + static_cast<size_t>(p.per) * 16);
  const TZ* zrow = z + row * p.ldz;
  TG* drow = GRAD ? dz + row * p.lddz : nullptr;

  long long target = -1;
  if (p.targets != nullptr) {
    target = p.targets[row];
    if (target >= p.vocab && rank == 0 && tid == 0) record_error(p.status, kErrBadIndex);
    if (target < 0 || target >= p.vocab) {  // the same for the whole cluster
      if (FORM != distill::kAgain && rank == 0 && tid == 0) p.loss[row] = 0.f;
      if (GRAD) zero_row(drow, p.dz_cols, rank * blockDim.x + tid, parts * blockDim.x);
      return;
    }
  }

  const Slice<TZ> s = rows::start_load(reinterpret_cast<TZ*>(smem), sh.bars, zrow, p.vocab, rank, p.per);
  if (warp == 0) {
    // The teacher's list and the student's logits at it, by every CTA for itself.
    float top = -CUDART_INF_F;
    int present = 0;
    bool has_target = false;
    for (int i = lane; i < p.k; i += 32) {
      long long c = p.ids64 ? static_cast<const long long*>(p.ids)[row * p.k + i]
                            : static_cast<const int*>(p.ids)[row * p.k + i];
      const float raw = teacher_logit(p, row * p.k + i) * p.inv_tau;
      if (c >= p.vocab) {
        if (rank == 0) record_error(p.status, kErrBadIndex);
        c = -1;
      }
      const float a = c < 0 ? -CUDART_INF_F : raw;
      list[i].col = c < 0 ? -1 : static_cast<int>(c);
      list[i].logp = a;
      list[i].z = c < 0 ? 0.f : to_f32(zrow[c]);
      top = fmaxf(top, a);
      present += c >= 0;
      has_target |= c >= 0 && c == target;
    }
    const float target_logit = p.ce != 0.f ? to_f32(zrow[target]) : 0.f;
    const float scale = distill::scale_of<FORM>(p, distill::scale_of_all(p), row);
    present = __reduce_add_sync(0xffffffffu, present);
    has_target = __any_sync(0xffffffffu, has_target);
    top = warp_max(top);
    // p_i = exp(a_i - base) / sum
    float base = 0.f, inv = 1.f, log_sum = 0.f;
    if (p.teacher_lse != nullptr) {
      base = p.teacher_lse[row];
    } else if (top != -CUDART_INF_F) {
      base = top;
      float e = 0.f;
      for (int i = lane; i < p.k; i += 32) e += expf(list[i].logp - base);
      e = warp_sum(e);
      inv = 1.f / e;
      log_sum = logf(e);
    }
    const bool empty = base == -CUDART_INF_F;  // the teacher's row has no logit at all: no mass, on the rest neither
    float mass = 0.f;
    for (int i = lane; i < p.k; i += 32) {
      const float a = empty ? -CUDART_INF_F : list[i].logp - base;
      list[i].logp = a - log_sum;
      list[i].p = expf(a) * inv;
      mass += list[i].p;
    }
    mass = warp_sum(mass);
    if (lane == 0) {
      const float rest = p.teacher_lse != nullptr && present > 0 && !empty ? 1.f - mass : 0.f;
      sh.mass = mass;
      sh.scale = scale;
      sh.rest = rest > kDistillLeastRest ? rest : 0.f;
      sh.target_logit = target_logit;
      sh.target_listed = has_target;
      sh.again = sh.repeats = sh.listed = 0;
    }
  }
  float mx = warp_max(rows::max_while_loading(s, sh.bars, p.status));
  if (lane == 0) sh.red_max[warp] = mx;
  __syncthreads();
  if (parts > 1) cluster.barrier_arrive();  // this CTA runs: its shared memory may be written
  mx = warp_max(lane < warps ? sh.red_max[lane] : -CUDART_INF_F);
  const float c = p.inv_tau * CUDART_L2E_F, c1 = POW == 1 ? CUDART_L2E_F : (POW > 1 ? POW : 1) * c;
  const rows::Ref ref(mx, c), ref1 = rows::ref_at_one<POW>(ref);

  // Take the listed logits out of the slice.  Entries that share a column agree on one: the slot holds the number
  // of its last writer until that one puts -inf there (no number has -inf's bits).
  for (int i = tid; i < p.k; i += blockDim.x)
    if (list[i].col >= 0 && s.holds(list[i].col)) put_mark(s.sm + (list[i].col - s.first), i);
  __syncthreads();
  for (int i = tid; i < p.k; i += blockDim.x) {
    const int col = list[i].col;
    bool owner = false;
    if (col >= 0 && s.holds(col)) {
      owner = get_mark(s.sm + (col - s.first)) == i;
      if (!owner) sh.repeats = 1;
      if (owner) s.sm[col - s.first] = rows::neg_inf<TZ>();
    }
    list[i].owner = owner;
    if (owner && p.k >= p.vocab) atomicAdd(&sh.listed, 1);  // only such a list can name every column
  }
  __syncthreads();
  const bool repeats = sh.repeats;
  if (parts > 1) cluster.barrier_wait();

  // sums over the slice and its listed columns, relative to the slice's largest logit
  {
    float2 acc[2] = {rows::both(0.f), rows::both(0.f)}, acc1[2] = {rows::both(0.f), rows::both(0.f)};
    rows::by_kind(ref, [&](auto far) {
      constexpr bool FAR = decltype(far)::value;
      const float2 c2 = rows::both(c), n2 = rows::both(FAR ? -ref.z : -ref.r);
      rows::for_vectors(s, [&](int v) {
        float2 q[E / 2];
        rows::load_pairs(s, v, q);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          const float2 e = rows::exp2_pair(rows::log2_pair<FAR>(q[i], c2, n2));
          acc[i & 1] = rows::add2(acc[i & 1], e);
          if constexpr (POW == 2) acc1[i & 1] = rows::fma2(e, e, acc1[i & 1]);
          if constexpr (POW == 1 || POW == 4)
            acc1[i & 1] = rows::add2(acc1[i & 1], rows::at_one<POW, FAR>(e, q[i], ref1));
        }
      });
    });
    float sum[4] = {(acc[0].x + acc[0].y) + (acc[1].x + acc[1].y), (acc1[0].x + acc1[0].y) + (acc1[1].x + acc1[1].y),
                    0.f, 0.f};
    if (repeats) {  // the first entry stands for a column, in every run
      for (int i = tid; i < p.k; i += blockDim.x)
        if (list[i].col >= 0 && s.holds(list[i].col)) list[i].owner = first_of_column(list, i);
    }
    for (int i = tid; i < p.k; i += blockDim.x) {
      if (list[i].owner) {
        sum[2] += exp2f(ref.log2_of(list[i].z, c));
        if (POW != 0) sum[3] += exp2f(ref1.log2_of(list[i].z, c1));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (POW == 0 && (i & 1)) continue;
      sum[i] = warp_sum(sum[i]);
      if (lane == 0) sh.red[warp][i] = sum[i];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (POW != 0 || !(i & 1)) sum[i] = warp_sum(lane < warps ? sh.red[lane][i] : 0.f);
      if (lane < parts) {
        Part* to = &(parts > 1 ? cluster.map_shared_rank(&sh, lane) : &sh)->part[rank];
        *to = Part{ref, ref1, sum[0], sum[1], sum[2], sum[3], sh.listed};
      }
      __syncwarp();
    }
  }
  if (parts > 1) cluster.sync();

  // The row's scalars, by the first warp of every CTA, the parts in the same order.
  rows::Ref top(0.f, c), top1 = rows::ref_at_one<POW>(top);
  float S = 0.f, total = 0.f, total1 = 0.f, m = 0.f;
  // What the gradient needs, and the loss, from the rest's sum relative to `at`, which is f (at temperature 1: f1) times the row's
  // reference, and the logarithm of the rest's probability.
  auto finish = [&](const rows::Ref& at, float f, float f1, float rest_sum, float log_rest) {
    const float scale = sh.scale;
    const float mass = sh.mass + m;
    const rows::Ref at1 = rows::ref_at_one<POW>(at);
    if (lane == 0) {
      float A = mass != 0.f ? mass * f / total : 0.f;
      if (m > 0.f && rest_sum > 0.f) A -= m / rest_sum;
      A *= scale * p.kd * p.tau;
      float B = p.ce != 0.f ? scale * p.ce * f1 / total1 : 0.f;
      if (POW == 0) {  // one exponential serves both terms
        A += B;
        B = 0.f;
      }
      sh.ref = at;
      sh.ref1 = at1;
      sh.A = A;
      sh.B = B;
      sh.top = top;
      sh.top1 = top1;
      sh.inv_sum = 1.f / total;
      sh.inv_sum1 = 1.f / total1;
      sh.all_mass = mass;
    }
    if (FORM != distill::kAgain && rank == 0) {
      const float log2_total = log2f(total);
      float kl = 0.f;
      for (int i = lane; i < p.k; i += 32) {
        const float logq = (top.log2_of(list[i].z, c) - log2_total) * CUDART_LN2_F;
        if (list[i].p != 0.f) kl += list[i].p * (list[i].logp - logq);
      }
      kl = warp_sum(kl);
      if (lane == 0) {
        if (m > 0.f) kl += m * (logf(m) - log_rest);
        float loss = p.kd != 0.f ? p.kd * p.tau * p.tau * kl : 0.f;
        if (p.ce != 0.f) loss += p.ce * (log2f(total1) - top1.log2_of(sh.target_logit, c1)) * CUDART_LN2_F;
        p.loss[row] = scale * loss;
      }
    }
  };
  if (warp == 0) {
    int best = -1, all_listed = 0;
    for (int q = 0; q < parts; ++q) {
      const Part& w = sh.part[q];
      if ((w.rest != 0.f || w.list != 0.f) && (best < 0 || w.ref.z > sh.part[best].ref.z)) best = q;
      all_listed += w.listed;
    }
    if (best >= 0) {
      top = sh.part[best].ref;
      top1 = sh.part[best].ref1;
    }
    float L = 0.f, S1 = 0.f, L1 = 0.f;
    for (int q = 0; q < parts; ++q) {
      const Part& w = sh.part[q];
      if (w.rest == 0.f && w.list == 0.f) continue;
      const float step = top.log2_of(w.ref, c), f = q == best ? 1.f : exp2f(step);
      S += w.rest * f;
      L += w.list * f;
      if (POW != 0) {
        const float f1 = q == best ? 1.f : exp2f(rows::log2_at_one<POW>(step, top1, w.ref1));
        S1 += w.rest1 * f1;
        L1 += w.list1 * f1;
      }
    }
    total = S + L;
    total1 = POW != 0 ? S1 + L1 : total;
    // a list that names every column leaves no rest, whatever rounding says
    m = p.k >= p.vocab && all_listed >= p.vocab ? 0.f : sh.rest;
    const bool again = m > 0.f && S < kLeastRestSum;
    if (lane == 0) sh.again = again;
    if (!again) finish(top, 1.f, 1.f, S, logf(S / total));
  }
  __syncthreads();
  if (sh.again) {  // the same for the whole cluster: the rest's sum, relative to the rest's own largest logit
    float rest_max = -CUDART_INF_F;
    for (int v = tid; v < s.nv; v += blockDim.x) {
      float e[E];
      load_vec<E>(s.sm + v * E, e);
#pragma unroll
      for (int i = 0; i < E; ++i) rest_max = fmaxf(rest_max, e[i]);
    }
    rest_max = warp_max(rest_max);
    if (lane == 0) sh.red_max[warp] = rest_max;
    __syncthreads();
    rest_max = warp_max(lane < warps ? sh.red_max[lane] : -CUDART_INF_F);
    const rows::Ref at(rest_max, c);
    float sum = 0.f;
    for (int v = tid; v < s.nv; v += blockDim.x) {
      float e[E];
      load_vec<E>(s.sm + v * E, e);
#pragma unroll
      for (int i = 0; i < E; ++i) sum += rows::fast_exp2(at.log2_of(e[i], c));
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.red[warp][0] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = warp_sum(lane < warps ? sh.red[lane][0] : 0.f);
      if (lane < parts) {
        Part* to = &(parts > 1 ? cluster.map_shared_rank(&sh, lane) : &sh)->again_part[rank];
        *to = Part{at, at, sum, 0.f, 0.f, 0.f, 0};
      }
      __syncwarp();
    }
    if (parts > 1) cluster.sync();
    if (warp == 0) {
      int best = -1;
      for (int q = 0; q < parts; ++q)
        if (sh.again_part[q].rest != 0.f && (best < 0 || sh.again_part[q].ref.z > sh.again_part[best].ref.z)) best = q;
      const rows::Ref own = best >= 0 ? sh.again_part[best].ref : top;  // else nothing finite outside the list
      S = 0.f;
      for (int q = 0; q < parts; ++q)
        if (sh.again_part[q].rest != 0.f) S += sh.again_part[q].rest * exp2f(own.log2_of(sh.again_part[q].ref, c));
      const float step = top.log2_of(own, c);
      finish(own, exp2f(step), exp2f(POW > 0 ? rows::log2_at_one<POW>(step, top1, rows::ref_at_one<POW>(own)) : step), S,
             logf(S) + top.log_of(own, c, p.inv_tau) - logf(total));
    }
    __syncthreads();
  }
  if (!GRAD) return;

  // gradient of the slice, then of the listed columns and the target
  const float A = sh.A, B = sh.B;
  const bool same_vectors =
      sizeof(TG) == sizeof(TZ)
          ? (reinterpret_cast<uintptr_t>(drow) & 15) / sizeof(TG) == static_cast<uintptr_t>(s.off)
          : s.off == 0 && (reinterpret_cast<uintptr_t>(drow) & (E * sizeof(TG) - 1)) == 0;
  const rows::Ref at = sh.ref, at1 = sh.ref1;
  const float2 A2 = rows::both(A), B2 = rows::both(B);
  rows::by_kind(at, [&](auto far) {
    constexpr bool FAR = decltype(far)::value;
    const float2 c2 = rows::both(c), n2 = rows::both(FAR ? -at.z : -at.r);
    rows::for_vectors(s, [&](int v) {
      float2 q[E / 2];
      rows::load_pairs(s, v, q);
      float g[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 e = rows::exp2_pair(rows::log2_pair<FAR>(q[i], c2, n2));
        float2 r;
        if constexpr (POW == 0)
          r = rows::mul2(e, A2);
        else if constexpr (POW == 2)
          r = rows::mul2(e, rows::fma2(e, B2, A2));
        else
          r = rows::fma2(rows::at_one<POW, FAR>(e, q[i], at1), B2, rows::mul2(e, A2));
        g[2 * i] = r.x;
        g[2 * i + 1] = r.y;
      }
      const int col = s.first + v * E;
      if (same_vectors && col >= 0 && col + E <= p.vocab) {
        store_vec<E>(drow + col, g);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (col + i >= 0 && col + i < p.vocab) drow[col + i] = from_f32<TG>(g[i]);
      }
    });
  });
  if (rank == parts - 1)
    for (int i = p.vocab + tid; i < p.dz_cols; i += blockDim.x) drow[i] = from_f32<TG>(0.f);
  __syncthreads();
  const float scale = sh.scale;
  const float kd = scale * p.kd * p.tau, ce = scale * p.ce;
  for (int i = tid; i < p.k; i += blockDim.x) {
    if (!list[i].owner) continue;
    const int col = list[i].col;
    float share = list[i].p;
    if (sh.repeats) {
      share = 0.f;
      for (int j = 0; j < p.k; ++j)
        if (list[j].col == col) share += list[j].p;
    }
    float g = kd != 0.f ? kd * (exp2f(sh.top.log2_of(list[i].z, c)) * sh.inv_sum * sh.all_mass - share) : 0.f;
    if (ce != 0.f) g += ce * (exp2f(sh.top1.log2_of(list[i].z, c1)) * sh.inv_sum1 - (col == target ? 1.f : 0.f));
    drow[col] = from_f32<TG>(g);
  }
  if (tid == 0 && ce != 0.f && !sh.target_listed && s.holds(static_cast<int>(target))) {
    const float v = to_f32(s.sm[target - s.first]);
    float g = rows::fast_exp2(at.log2_of(v, c)) * A - ce;
    if (POW != 0) g += rows::fast_exp2(at1.log2_of(v, c1)) * B;
    drow[target] = from_f32<TG>(g);
  }
}

// Row r of dz times g[r * gstep].  Rows whose factor is 1 are not touched, so the usual call, whose scale was
// applied when dz was formed, reads the factors and leaves.
template <typename T>
__global__ void __launch_bounds__(256) scale_in_place_kernel(T* __restrict__ dz, long long rows, int cols,
                                                             long long ld, const float* __restrict__ g, int gstep) {
  if (gstep == 0 && *g == 1.f) return;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float f = g[r * gstep];
    if (f == 1.f) continue;
    T* row = dz + r * ld;
    for (int c = threadIdx.x; c < cols; c += 256) row[c] = from_f32<T>(to_f32(row[c]) * f);
  }
}

}  // namespace

void distill_loss(const DistillArgs& a, cudaStream_t stream) {
  TTB_CHECK(a.k >= 1 && a.k <= kDistillMaxList, "distillation: between 1 and 1024 listed columns");
  TTB_CHECK(a.vocab >= 1 && logits_row_fits(a.vocab, a.z_type), "distillation: the rows are too long");
  TTB_CHECK(a.tau > 0.f, "distillation: the temperature must be positive");
  TTB_CHECK(a.dz == nullptr || a.dz_cols >= a.vocab, "distillation: the gradient has too few columns");
  TTB_CHECK(a.dz == nullptr || a.dz_type == a.z_type ||
                (a.z_type == ScalarType::kF32 && a.dz_type == ScalarType::kBF16),
            "distillation: the gradient has the logits' type, or bf16 for fp32 logits");
  TTB_CHECK(a.factor == nullptr || (a.dz != nullptr && a.z_type == ScalarType::kF16 && a.dz_type == a.z_type),
            "distillation: factors multiply an fp16 gradient");
  if (a.rows == 0) return;
  const rows::Plan plan = rows::plan_rows(a.rows, a.vocab, scalar_bytes(a.z_type));
  TTB_CHECK(a.rows * plan.parts <= 0x7FFFFFFFLL, "distillation: too many rows");
  Params p{};
  p.vocab = a.vocab;
  p.k = a.k;
  p.per = plan.per;
  p.parts = plan.parts;
  p.dz_cols = a.dz_cols;
  p.ids64 = a.ids64;
  p.inv_tau = 1.f / a.tau;
  p.tau = a.tau;
  p.kd = a.kd;
  p.ce = a.ce;
  p.ids = a.ids;
  p.t = a.t;
  p.t_type = a.t_type;
  p.teacher_lse = a.teacher_lse;
  p.targets = a.targets;
  p.scale = a.scale;
  p.factor = a.factor;
  p.factor_step = a.factor_step;
  p.loss = a.loss;
  p.ldz = a.ldz;
  p.lddz = a.lddz;
  p.status = a.status;
  const int pow = a.ce == 0.f || a.tau == 1.f ? 0 : a.tau == 2.f ? 2 : a.tau == 4.f ? 4 : 1;
  if (distill::loss_by_ring(a, p, pow, stream)) return;
  const size_t smem = plan.slice_bytes + a.k * sizeof(Entry);
  auto launch = [&](auto kernel, auto* z, auto* dz) {
    TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows * plan.parts));
    cfg.blockDim = dim3(plan.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = plan.parts > 1 ? 1 : 0;
    TTB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, z, dz, p));
  };
  distill::with_kernel_types(a, [&](const auto* z, auto* dz) {
    using TZ = std::remove_const_t<std::remove_pointer_t<decltype(z)>>;
    using TG = std::remove_pointer_t<decltype(dz)>;
    distill::with_pow(pow, [&](auto w) {
      constexpr int POW = decltype(w)::value;
      distill::with_form<TZ, TG>(a, [&](auto form) { launch(distill_kernel<TZ, TG, decltype(form)::value, POW>, z, dz); });
    });
  });
}

void scale_in_place(void* dz, ScalarType type, long long rows, int cols, long long ld, const float* g, int gstep,
                    cudaStream_t stream) {
  if (rows == 0) return;
  const long long most = 8LL * num_sms();
  with_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    scale_in_place_kernel<T><<<static_cast<int>(rows < most ? rows : most), 256, 0, stream>>>(
        static_cast<T*>(dz), rows, cols, ld, g, gstep);
  });
  TTB_CUDA_CHECK(cudaGetLastError());
}

}  // namespace ttb
