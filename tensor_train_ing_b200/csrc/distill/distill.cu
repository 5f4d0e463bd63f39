// Distillation from a teacher's top logits: the loss of every row and, in the same pass over the logits, its
// gradient (formulas in distill_api.h).
//
// A row sits in the shared memory of a cluster (row_slice.cuh), so the gradient needs no second read of
// it.  The listed columns are taken out of the slice first (replaced by -inf): what the passes over the slice
// then sum is the rest of the row, whose mass q_rest is thereby never the difference of two nearly equal
// numbers.  With M the largest unlisted logit, every unlisted column's gradient is
//     exp((z_j - M) / tau) A + exp(z_j - M) B,
//     A = scale kd tau ((P + m) exp(M / tau - lse_tau) - m / S),  S = sum over the rest of exp((z - M) / tau)
//     B = scale ce exp(M - lse_1)
// which overflows nowhere; the few listed columns and the target are written after the others.
#include "../common/host.h"
#include "distill_api.h"
#include "row_slice.cuh"

namespace ttb {
namespace {

using rows::Slice;
namespace cg = cooperative_groups;

struct Part {  // what one CTA knows of its slice; sums are relative to the maxima
  float rest_max, rest_sum, rest_sum1;  // unlisted columns, at tau and at 1
  float list_max, list_sum, list_sum1;  // listed columns (each counted once)
  int listed;
};

struct Shared {
  Part part[rows::kMaxParts];
  float red[32][4];
  float target_logit;
  float mass, rest;  // P and m
  int entries;       // present entries of the list
  // the row's scalars for the gradient: q_j = exp((z_j - top) / tau) inv_sum
  float ref, A, B, top, inv_sum, inv_sum1, all_mass;
};

struct Params {
  int vocab, k, per, dz_cols;
  bool ids64;
  float inv_tau, tau, kd, ce;
  const void* ids;
  const float* teacher_lse;
  const long long* targets;
  const float* scale;
  float* loss;
  long long ldz, lddz;
  uint32_t* status;
};

template <int N>
__device__ __forceinline__ void block_reduce_max(float (&v)[N], float (*red)[4]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_max(v[i]);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[threadIdx.x >> 5][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = red[0][i];
    for (int w = 1; w < blockDim.x / 32; ++w) v[i] = fmaxf(v[i], red[w][i]);
  }
  __syncthreads();
}
template <int N>
__device__ __forceinline__ void block_reduce_sum(float (&v)[N], float (*red)[4]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[threadIdx.x >> 5][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = red[0][i];
    for (int w = 1; w < blockDim.x / 32; ++w) v[i] += red[w][i];
  }
  __syncthreads();
}

// Entry i of the shared-memory copy of the teacher's list.
struct Entry {
  int col;      // -1: absent
  float logp, p;  // log p_i and p_i (0: no mass)
  float z;      // the student's logit at col
  int owner;    // whether this entry stands for its column here (the first CTA-local entry with this column)
};

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

// TWO: cross-entropy at another temperature than the divergence's, which needs a second exponential.
template <typename TZ, typename TT, typename TG, bool GRAD, bool TWO>
__global__ void __launch_bounds__(512) distill_kernel(const TZ* __restrict__ z, const TT* __restrict__ t,
                                                      TG* __restrict__ dz, const __grid_constant__ Params p) {
  constexpr int E = Slice<TZ>::kVec;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), rank = cluster.block_rank();
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto* list = reinterpret_cast<Entry*>(smem + static_cast<size_t>(p.per) * 16);
  const TZ* zrow = z + row * p.ldz;
  TG* drow = GRAD ? dz + row * p.lddz : nullptr;

  long long target = -1;
  bool live = true;
  if (p.targets != nullptr) {
    target = p.targets[row];
    if (target >= p.vocab) {
      if (rank == 0 && tid == 0) record_error(p.status, kErrBadIndex);
      target = -1;
    }
    live = target >= 0;
  }
  if (!live) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) p.loss[row] = 0.f;
    if (GRAD)
      for (int c = rank * blockDim.x + tid; c < p.dz_cols; c += parts * blockDim.x) drow[c] = from_f32<TG>(0.f);
    return;
  }

  const Slice<TZ> s = rows::start_load(reinterpret_cast<TZ*>(smem), zrow, p.vocab, rank, p.per);

  // the teacher's list, by the first warp of every CTA, while the row arrives
  if (warp == 0) {
    float top = -CUDART_INF_F;
    int present = 0;
    for (int i = lane; i < p.k; i += 32) {
      long long c = p.ids64 ? static_cast<const long long*>(p.ids)[row * p.k + i]
                            : static_cast<const int*>(p.ids)[row * p.k + i];
      if (c >= p.vocab) {
        if (rank == 0) record_error(p.status, kErrBadIndex);
        c = -1;
      }
      const float a = c < 0 ? -CUDART_INF_F : to_f32(t[row * p.k + i]) * p.inv_tau;
      list[i].col = c < 0 ? -1 : static_cast<int>(c);
      list[i].logp = a;
      list[i].z = 0.f;
      list[i].owner = 0;
      top = fmaxf(top, a);
      present += c >= 0;
    }
    present = __reduce_add_sync(0xffffffffu, present);
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
    float mass = 0.f;
    for (int i = lane; i < p.k; i += 32) {
      const float a = list[i].logp - base;
      list[i].logp = a - log_sum;
      list[i].p = expf(a) * inv;
      mass += list[i].p;
    }
    mass = warp_sum(mass);
    if (lane == 0) {
      const float rest = p.teacher_lse != nullptr && present > 0 ? 1.f - mass : 0.f;
      sh.mass = mass;
      sh.rest = rest > kDistillLeastRest ? rest : 0.f;
      sh.entries = present;
    }
  }
  rows::finish_load();
  if (parts > 1) cluster.sync();  // every CTA of the row runs: its shared memory may be written

  // Take the listed logits out of the slice: read them, let the entries that share a column agree on one (the
  // slot holds the number of the last writer), then put -inf.  The first CTA gets a copy of all of them.
  Entry* first_list = cluster.map_shared_rank(list, 0);
  for (int i = tid; i < p.k; i += blockDim.x) {
    const int c = list[i].col;
    if (c >= 0 && s.holds(c)) {
      const float v = to_f32(s.sm[c - s.first]);
      list[i].z = v;
      if (rank != 0) first_list[i].z = v;
    }
  }
  if (tid == 0 && target >= 0 && s.holds(static_cast<int>(target)))
    cluster.map_shared_rank(&sh, 0)->target_logit = to_f32(s.sm[target - s.first]);
  __syncthreads();
  for (int i = tid; i < p.k; i += blockDim.x)
    if (list[i].col >= 0 && s.holds(list[i].col)) put_mark(s.sm + (list[i].col - s.first), i);
  __syncthreads();
  bool shared_column = false;
  bool target_listed = false;
  for (int i = tid; i < p.k; i += blockDim.x) {
    const int c = list[i].col;
    if (c >= 0 && s.holds(c)) {
      list[i].owner = get_mark(s.sm + (c - s.first)) == i;
      shared_column |= !list[i].owner;
    }
    target_listed |= c >= 0 && c == target;
  }
  const bool repeats = __syncthreads_or(shared_column);
  target_listed = __syncthreads_or(target_listed);
  float list_max = -CUDART_INF_F;
  int listed = 0;
  for (int i = tid; i < p.k; i += blockDim.x) {
    if (list[i].owner) {
      s.sm[list[i].col - s.first] = rows::neg_inf<TZ>();
      list_max = fmaxf(list_max, list[i].z);
      ++listed;
    }
  }
  __syncthreads();

  // the slice's maxima and sums
  float mx[2] = {-CUDART_INF_F, list_max};
  for (int v = tid; v < s.nv; v += blockDim.x) {
    float e[E];
    load_vec<E>(s.sm + v * E, e);
#pragma unroll
    for (int i = 0; i < E; ++i) mx[0] = fmaxf(mx[0], e[i]);
  }
  block_reduce_max(mx, sh.red);
  const float c2 = p.inv_tau * CUDART_L2E_F;
  float ref = isfinite(mx[0]) ? mx[0] : 0.f;
  const float list_ref = isfinite(mx[1]) ? mx[1] : 0.f;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int v = tid; v < s.nv; v += blockDim.x) {
    float e[E];
    load_vec<E>(s.sm + v * E, e);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float x = e[i] - ref;
      sum[0] += rows::fast_exp2(x * c2);
      if (TWO) sum[1] += rows::fast_exp2(x * CUDART_L2E_F);
    }
  }
  for (int i = tid; i < p.k; i += blockDim.x) {
    if (list[i].owner) {
      const float x = list[i].z - list_ref;
      sum[2] += expf(x * p.inv_tau);
      if (TWO) sum[3] += expf(x);
    }
  }
  block_reduce_sum(sum, sh.red);
  int owned = 0;  // only a list as long as the row can name every column
  if (p.k >= p.vocab) {
    float n[1] = {static_cast<float>(listed)};
    block_reduce_sum(n, sh.red);
    owned = static_cast<int>(n[0]);
  }
  if (tid < parts) {
    Part* q = &cluster.map_shared_rank(&sh, tid)->part[rank];
    *q = Part{mx[0], sum[0], sum[1], mx[1], sum[2], sum[3], owned};
  }
  if (parts > 1)
    cluster.sync();
  else
    __syncthreads();

  if (warp == 0) {
    // every CTA combines the parts in the same order
    float rest_max = -CUDART_INF_F, lmax = -CUDART_INF_F;
    int all_listed = 0;
    for (int c = 0; c < parts; ++c) {
      rest_max = fmaxf(rest_max, sh.part[c].rest_max);
      lmax = fmaxf(lmax, sh.part[c].list_max);
      all_listed += sh.part[c].listed;
    }
    const float row_ref = isfinite(rest_max) ? rest_max : 0.f;
    const float lref = isfinite(lmax) ? lmax : 0.f;
    float S = 0.f, S1 = 0.f, L = 0.f, L1 = 0.f;
    for (int c = 0; c < parts; ++c) {
      const Part& q = sh.part[c];
      const float dr = (isfinite(q.rest_max) ? q.rest_max : 0.f) - row_ref;
      const float dl = (isfinite(q.list_max) ? q.list_max : 0.f) - lref;
      if (q.rest_sum != 0.f) S += q.rest_sum * expf(dr * p.inv_tau);
      if (q.list_sum != 0.f) L += q.list_sum * expf(dl * p.inv_tau);
      if (TWO) {
        if (q.rest_sum1 != 0.f) S1 += q.rest_sum1 * expf(dr);
        if (q.list_sum1 != 0.f) L1 += q.list_sum1 * expf(dl);
      }
    }
    // The row's sums relative to its largest logit: probabilities come from these, not from a log-sum-exp,
    // whose rounding (half an ulp of a number around 10) would enter every one of them.
    const float hi = fmaxf(rest_max, lmax);
    const float top = isfinite(hi) ? hi : 0.f;
    const float fr = S != 0.f ? expf((row_ref - top) * p.inv_tau) : 0.f;
    const float total = S * fr + (L != 0.f ? L * expf((lref - top) * p.inv_tau) : 0.f);
    float fr1 = fr, total1 = total;
    if (TWO) {
      fr1 = S1 != 0.f ? expf(row_ref - top) : 0.f;
      total1 = S1 * fr1 + (L1 != 0.f ? L1 * expf(lref - top) : 0.f);
    }
    const float scale = p.scale != nullptr ? *p.scale : 1.f;
    // a list that names every column leaves no rest, whatever rounding says
    const float m = p.k >= p.vocab && all_listed >= p.vocab ? 0.f : sh.rest;
    const float mass = sh.mass + m;
    if (lane == 0) {
      sh.ref = row_ref;
      sh.top = top;
      sh.inv_sum = 1.f / total;
      sh.inv_sum1 = 1.f / total1;
      sh.all_mass = mass;
      float A = mass != 0.f ? mass * fr / total : 0.f;
      if (m > 0.f && S > 0.f) A -= m / S;
      A *= scale * p.kd * p.tau;
      float B = p.ce != 0.f ? scale * p.ce * fr1 / total1 : 0.f;
      if (!TWO) {
        A += B;
        B = 0.f;
      }
      sh.A = A;
      sh.B = B;
    }
    if (rank == 0) {
      float kl = 0.f;
      for (int i = lane; i < p.k; i += 32) {
        const float logq = (list[i].z - top) * p.inv_tau - logf(total);
        if (list[i].p != 0.f) kl += list[i].p * (list[i].logp - logq);
      }
      kl = warp_sum(kl);
      if (lane == 0) {
        if (m > 0.f)  // log q_rest from its parts where the probability itself leaves fp32's range
          kl += m * (fr > 1e-30f ? logf(m / (S * fr / total))
                                 : logf(m) - (logf(S) + (row_ref - top) * p.inv_tau - logf(total)));
        float loss = p.kd != 0.f ? p.kd * p.tau * p.tau * kl : 0.f;
        if (p.ce != 0.f) loss += p.ce * (logf(total1) - (sh.target_logit - top));
        p.loss[row] = scale * loss;
      }
    }
  }
  if (!GRAD) return;
  __syncthreads();

  // gradient of the slice, then of the listed columns and the target
  ref = sh.ref;
  const float A = sh.A, B = sh.B;
  const bool same_vectors =
      sizeof(TG) == sizeof(TZ)
          ? (reinterpret_cast<uintptr_t>(drow) & 15) / sizeof(TG) == static_cast<uintptr_t>(s.off)
          : s.off == 0 && (reinterpret_cast<uintptr_t>(drow) & (E * sizeof(TG) - 1)) == 0;
  for (int v = tid; v < s.nv; v += blockDim.x) {
    float e[E];
    load_vec<E>(s.sm + v * E, e);
    const int col = s.first + v * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float x = e[i] - ref;
      e[i] = rows::fast_exp2(x * c2) * A;
      if (TWO) e[i] += rows::fast_exp2(x * CUDART_L2E_F) * B;
    }
    if (same_vectors && col >= 0 && col + E <= p.vocab) {
      store_vec<E>(drow + col, e);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (col + i >= 0 && col + i < p.vocab) drow[col + i] = from_f32<TG>(e[i]);
    }
  }
  if (rank == parts - 1)
    for (int c = p.vocab + tid; c < p.dz_cols; c += blockDim.x) drow[c] = from_f32<TG>(0.f);
  __syncthreads();
  const float scale = p.scale != nullptr ? *p.scale : 1.f;
  const float kd = scale * p.kd * p.tau, ce = scale * p.ce;
  for (int i = tid; i < p.k; i += blockDim.x) {
    if (!list[i].owner) continue;
    const int c = list[i].col;
    float share = list[i].p;
    if (repeats) {
      share = 0.f;
      for (int j = 0; j < p.k; ++j)
        if (list[j].col == c) share += list[j].p;
    }
    float g = kd != 0.f ? kd * (expf((list[i].z - sh.top) * p.inv_tau) * sh.inv_sum * sh.all_mass - share) : 0.f;
    if (ce != 0.f) g += ce * (expf(list[i].z - sh.top) * sh.inv_sum1 - (c == target ? 1.f : 0.f));
    drow[c] = from_f32<TG>(g);
  }
  if (tid == 0 && ce != 0.f && target >= 0 && !target_listed && s.holds(static_cast<int>(target))) {
    const float x = to_f32(s.sm[target - s.first]) - ref;
    float g = rows::fast_exp2(x * c2) * A - ce;
    if (TWO) g += rows::fast_exp2(x * CUDART_L2E_F) * B;
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
  if (a.rows == 0) return;
  const rows::Plan plan = rows::plan_rows(a.rows, a.vocab, scalar_bytes(a.z_type));
  TTB_CHECK(a.rows * plan.parts <= 0x7FFFFFFFLL, "distillation: too many rows");
  Params p{};
  p.vocab = a.vocab;
  p.k = a.k;
  p.per = plan.per;
  p.dz_cols = a.dz_cols;
  p.ids64 = a.ids64;
  p.inv_tau = 1.f / a.tau;
  p.tau = a.tau;
  p.kd = a.kd;
  p.ce = a.ce;
  p.ids = a.ids;
  p.teacher_lse = a.teacher_lse;
  p.targets = a.targets;
  p.scale = a.scale;
  p.loss = a.loss;
  p.ldz = a.ldz;
  p.lddz = a.lddz;
  p.status = a.status;
  const bool two = a.ce != 0.f && a.tau != 1.f;
  const size_t smem = plan.slice_bytes + a.k * sizeof(Entry);
  auto launch = [&](auto kernel, auto* z, auto* t, auto* dz) {
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
    cfg.numAttrs = 1;
    TTB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, z, t, dz, p));
  };
  with_type(a.z_type, [&](auto* tz) {
    using TZ = std::remove_pointer_t<decltype(tz)>;
    with_type(a.t_type, [&](auto* tt) {
      using TT = std::remove_pointer_t<decltype(tt)>;
      auto with_grad = [&](auto* tg) {
        using TG = std::remove_pointer_t<decltype(tg)>;
        const auto* zp = static_cast<const TZ*>(a.z);
        const auto* tp = static_cast<const TT*>(a.t);
        auto* gp = static_cast<TG*>(a.dz);
        if (gp == nullptr)
          two ? launch(distill_kernel<TZ, TT, TG, false, true>, zp, tp, gp)
              : launch(distill_kernel<TZ, TT, TG, false, false>, zp, tp, gp);
        else
          two ? launch(distill_kernel<TZ, TT, TG, true, true>, zp, tp, gp)
              : launch(distill_kernel<TZ, TT, TG, true, false>, zp, tp, gp);
      };
      if (a.dz != nullptr && a.dz_type != a.z_type)
        with_grad(static_cast<__nv_bfloat16*>(nullptr));
      else
        with_grad(static_cast<TZ*>(nullptr));
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
