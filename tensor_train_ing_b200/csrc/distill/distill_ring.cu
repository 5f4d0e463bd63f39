// The distillation loss of many long rows: a persistent kernel of CTAs, or of clusters that share a row, whose warps have
// roles, so that no step of a row waits for another row's memory latency.
//
//   consumers  sum the row as it arrives, then (gradient) write exp((z - R) / tau) A + exp(z - R) B over it
//   producer   keeps the row's stages coming: a stage of the next row as soon as the consumers are done with it
//   lister     reads the teacher's list of the next row, and the student's logits at it, while this row is worked on
//   patcher    takes the listed columns out of each stage as it arrives (replaces them by -inf)
//   finisher   turns the sums into the loss and the gradient's scalars, and writes the listed columns' gradient
//
// What they hand over is kept for several rows; every hand-over is an mbarrier with bounded waits, and a wait that runs
// out ends all roles.  The arithmetic is that of distill.cu, of which this is the form for long rows: 4096 rows of 50257
// bf16 logits, the loss alone, took 142 us there, with two CTAs of an SM each waiting through about 6 us of latencies per
// row, and 92 us here (63 us for the bytes); loss and gradient of 8192 rows at tau 2 took 422 us and 333 us (252 us).  4096 rows
// of 131072 fp32 logits, in clusters: 903 us (658 us).  8192 rows of 50257 fp32 logits with a bf16 gradient: 471 us (378 us).  No
// unit is full (special functions and issue slots 50 to 57 %, DRAM 48 to 55 %): the twelve consumer warps of a CTA are each in a
// chain of one vector's load, exponentials and sums.
#include <map>
#include <mutex>
#include <tuple>

#include "../common/host.h"
#include "distill_common.cuh"
#include "row_ring.cuh"

namespace ttb {
namespace distill {
namespace {

using rows::Ref;
using rows::Span;
using rows::kRingThreads;
using rows::kRingWarps;
using rows::kStages;
using rows::wait_for;
using rows::warp_arrives;
using rows::warp_waits;

constexpr int kThreads = 512;
constexpr int kProducer = kRingWarps, kLister = kRingWarps + 1, kPatcher = kRingWarps + 2, kFinisher = kRingWarps + 3;
static_assert(kFinisher == kThreads / 32 - 1);
// Rows that are between their list and their end at one time: the lister runs up to three rows ahead, which covers its two
// dependent reads of global memory and the finisher's turn before them.
constexpr int kSides = 4;

struct Listed {
  int col;        // -1: absent
  float logp, p;  // log p_i and p_i (0: no mass)
  float z;        // the student's logit at col
  short stage;    // that brings col; kStages: an edge column, -1: none
  short owner;    // the one entry that stands for its column
};

struct Row {  // what the lister says about a row
  long long row;  // -1: no more rows
  int live, target;
  float mass, rest, target_logit, list_top;
  unsigned edges;  // listed edge columns, by slot
  float edge[16];  // the edge columns' logits, by slot
  int first;       // column of the slice's first element
  int repeats, target_listed;
  int target_here;  // the CTA has the target's column
};

struct Scalars {
  float at, A, B;
};

struct Part {  // what one CTA of the row's knows of its columns: sums at tau and at 1
  float ref;          // the reference logit of the unlisted columns' sums (-inf: none)
  float sum, sum1;
  float list, list1;  // of the listed columns, each once, relative to the largest listed logit of the row
};

struct Shared {
  uint64_t full[kStages], ready[kStages], empty[kStages];
  uint64_t list_ready[kSides], side_free[kSides], sums_ready[kSides], scalars_ready[kSides], gradient_done[kSides];
  uint64_t part_ready[2];
  Row row[kSides];
  Scalars scalars[kSides];
  Part part[2][rows::kMaxParts];
  rows::WarpSum sums[kSides][kRingWarps];
  int stop;
};

// The row's CTA this one is, and the rows its cluster takes.
struct Place {
  int rank;
  long long row0, step;
};

__device__ __forceinline__ bool counts(const Params& p, long long row, long long& target) {
  target = p.targets != nullptr ? p.targets[row] : 0;
  return target >= 0 && target < p.vocab;
}

template <typename TZ>
__device__ __forceinline__ void produce(const TZ* z, TZ* sm, Shared& sh, const Params& p, const Place& at) {
  long long target;
  bool live = at.row0 < p.rows && counts(p, at.row0, target);
  int turn = 0;
  bool ok = true;
  for (long long row = at.row0; row < p.rows && ok; row += at.step) {
    const bool now = live;
    if (row + at.step < p.rows) live = counts(p, row + at.step, target);
    if (!now) continue;
    const Span<TZ> s(z + row * p.ldz, p.vocab, at.rank, p.per);
    for (int g = 0; g < kStages && ok; ++g) {
      if (turn > 0) ok = wait_for(&sh.empty[g], (turn - 1) & 1, &sh.stop, p.status);
      if (ok) s.load_stage(sm, sh.full, g);
    }
    ++turn;
  }
  if (!ok)  // copies under way end before the CTA does
    for (int g = 0; g < kStages; ++g)
      if (turn > 0) mbar_wait(&sh.full[g], (turn - 1) & 1, p.status, kErrTimeoutProducer);
}

template <typename TZ>
__device__ __forceinline__ void list_rows(const TZ* z, Listed* lists, Shared& sh, const Params& p, const Place& at) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (long long row = at.row0;; row += at.step, ++n) {
    const int side = n % kSides;
    if (n >= kSides && !warp_waits(&sh.side_free[side], (n / kSides - 1) & 1, &sh.stop, p.status)) return;
    Row& r = sh.row[side];
    if (row >= p.rows) {
      if (lane == 0) r.row = -1;
      warp_arrives(&sh.list_ready[side]);
      return;
    }
    long long target;
    const bool live = counts(p, row, target);
    if (!live) {
      if (lane == 0) {
        if (target >= p.vocab && at.rank == 0) record_error(p.status, kErrBadIndex);
        r.row = row;
        r.live = 0;
      }
      warp_arrives(&sh.list_ready[side]);
      continue;
    }
    if (p.targets == nullptr) target = -1;
    const Span<TZ> s(z + row * p.ldz, p.vocab, at.rank, p.per);
    Listed* list = lists + side * p.k;
    float top = -CUDART_INF_F, list_top = -CUDART_INF_F;
    bool present = false, has_target = false;
    for (int i = lane; i < p.k; i += 32) {
      long long col = p.ids64 ? static_cast<const long long*>(p.ids)[row * p.k + i]
                              : static_cast<const int*>(p.ids)[row * p.k + i];
      const float a = teacher_logit(p, row * p.k + i) * p.inv_tau;
      if (col >= p.vocab) {
        if (at.rank == 0) record_error(p.status, kErrBadIndex);
        col = -1;
      }
      Listed e;
      e.col = col < 0 ? -1 : static_cast<int>(col);
      e.logp = col < 0 ? -CUDART_INF_F : a;
      e.p = 0.f;
      e.z = col < 0 ? 0.f : to_f32(s.row[col]);
      e.stage = col < 0 || !s.holds(e.col) ? -1 : s.stage_of(e.col);
      e.owner = 0;
      list[i] = e;
      top = fmaxf(top, e.logp);
      if (col >= 0) list_top = fmaxf(list_top, e.z);
      present |= col >= 0;
      has_target |= col >= 0 && col == target;
    }
    const float target_logit = p.ce != 0.f ? to_f32(s.row[target]) : 0.f;
    const int edge = lane < 16 ? s.edge_column(lane) : -1;
    if (edge >= 0) r.edge[lane] = to_f32(s.row[edge]);
    present = __any_sync(0xffffffffu, present);
    has_target = __any_sync(0xffffffffu, has_target);
    top = warp_max(top);
    list_top = warp_max(list_top);
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
      const float rest = p.teacher_lse != nullptr && present && !empty ? 1.f - mass : 0.f;
      r.row = row;
      r.live = 1;
      r.target = static_cast<int>(target);
      r.mass = mass;
      r.rest = rest > kDistillLeastRest ? rest : 0.f;
      r.target_logit = target_logit;
      r.list_top = fabsf(list_top) < CUDART_INF_F ? list_top : 0.f;
      r.edges = 0u;
      r.first = s.first;
      r.repeats = 0;
      r.target_listed = has_target;
      r.target_here = target >= 0 && s.holds(static_cast<int>(target));
    }
    __syncwarp();
    for (int i = lane; i < p.k; i += 32) {  // edge columns are never in shared memory: they are settled here
      if (list[i].stage != kStages) continue;
      const unsigned bit = 1u << s.edge_slot(list[i].col);
      const bool owner = !(atomicOr(&r.edges, bit) & bit);
      list[i].owner = owner;
      if (!owner) r.repeats = 1;
    }
    warp_arrives(&sh.list_ready[side]);
  }
}

template <typename TZ>
__device__ __forceinline__ void patch_stages(TZ* sm, Listed* lists, Shared& sh, const Params& p) {
  const int lane = threadIdx.x & 31;
  int turn = 0;
  for (int n = 0;; ++n) {
    const int side = n % kSides;
    if (!warp_waits(&sh.list_ready[side], (n / kSides) & 1, &sh.stop, p.status)) return;
    Row& r = sh.row[side];
    if (r.row < 0) return;
    Listed* list = lists + side * p.k;
    for (int g = 0; g < kStages && r.live; ++g) {
      if (!warp_waits(&sh.full[g], turn & 1, &sh.stop, p.status)) return;
      // Entries that share a column agree on one: the slot holds the number of its last writer until that one puts
      // -inf there (no number has -inf's bits).  Element e of the row lies at e + off from the slice's start.
      for (int i = lane; i < p.k; i += 32)
        if (list[i].stage == g) put_mark(sm + list[i].col - r.first, i);
      __syncwarp();
      for (int i = lane; i < p.k; i += 32) {
        if (list[i].stage != g) continue;
        TZ* slot = sm + list[i].col - r.first;
        const bool owner = get_mark(slot) == i;
        list[i].owner = owner;
        if (owner)
          *slot = rows::neg_inf<TZ>();
        else
          r.repeats = 1;
      }
      fence_proxy_async_smem();  // before the stage's next copy
      warp_arrives(&sh.ready[g]);
    }
    turn += r.live;
    warp_arrives(&sh.side_free[side]);
  }
}

template <typename TZ, typename TG, int FORM, int POW>
__device__ __forceinline__ void consume(const TZ* z, TG* dz, const TZ* sm, const Listed* lists, Shared& sh,
                                        const Params& p, const Place& at, float c) {
  constexpr int E = Span<TZ>::kVec;
  constexpr bool GRAD = FORM != kLoss;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int turn = 0;
  unsigned on_side = 0;  // bit s: the parity of the live rows side s has had
  for (int n = 0;; ++n) {
    const int side = n % kSides;
    if (!warp_waits(&sh.list_ready[side], (n / kSides) & 1, &sh.stop, p.status)) return;
    const long long row = sh.row[side].row;
    if (row < 0) return;
    TG* drow = GRAD ? dz + row * p.lddz : nullptr;
    if (!sh.row[side].live) {
      if (GRAD) zero_row(drow, p.dz_cols, at.rank * kRingThreads + tid, p.parts * kRingThreads);
      warp_arrives(&sh.sums_ready[side]);
      continue;
    }
    const Span<TZ> s(z + row * p.ldz, p.vocab, at.rank, p.per);
    const int edge = tid < 16 ? s.edge_column(tid) : -1;
    const float edge_z = edge >= 0 ? sh.row[side].edge[tid] : 0.f;

    rows::Sums<POW> sums(c);
    bool sure = false;  // all threads of the warp have a reference: vectors are added without looking for one
#pragma unroll 1
    for (int g = 0; g < kStages; ++g) {
      if (!warp_waits(&sh.ready[g], turn & 1, &sh.stop, p.status)) return;
      if (sure) {
        s.for_stage(sm, g, [&](const uint4& u, int) { sums.template add_vector<TZ, false>(u, c); });
      } else {
        s.for_stage(sm, g, [&](const uint4& u, int) {
          sums.see(rows::max_of<TZ>(u), c);
          sums.template add_seen<TZ>(u, c);
        });
        sure = sums.settle(c);
      }
      if (!GRAD) warp_arrives(&sh.empty[g]);
    }
    const bool counted = edge >= 0 && !((sh.row[side].edges >> tid) & 1u);
    if (counted) sums.add_one(edge_z, c);
    if (sums.overflowed()) {  // rare: logits 40 tau above a thread's first ones, infinities, NaN
      const Listed* list = lists + side * p.k;
      sums = rows::Sums<POW>(c);
      for (int v = tid < s.lo ? tid + kRingThreads : tid; v < s.hi; v += kRingThreads) {
        const int col = s.first + v * E;
        unsigned out = 0;  // bit e: element e is listed
        for (int i = 0; i < p.k; ++i)
          if (const unsigned e = list[i].col - col; e < E) out |= 1u << e;
        for (int e = 0; e < E; ++e)
          if (!((out >> e) & 1u)) sums.add_one(to_f32(s.row[col + e]), c);
      }
      if (counted) sums.add_one(edge_z, c);
    }
    const rows::WarpSum mine = rows::warp_total<POW>(sums, c);
    if (lane == 0) sh.sums[side][warp] = mine;
    warp_arrives(&sh.sums_ready[side]);

    if (GRAD) {
      if (!warp_waits(&sh.scalars_ready[side], (on_side >> side) & 1, &sh.stop, p.status)) return;
      const Scalars k = sh.scalars[side];
      const Ref from(k.at, c), from1 = rows::ref_at_one<POW>(from);
      const auto gradient = [&](float2 q, auto far) {
        constexpr bool FAR = decltype(far)::value;
        const float2 e = rows::exp2_pair(rows::log2_pair<FAR>(q, rows::both(c), rows::both(FAR ? -from.z : -from.r)));
        if constexpr (POW == 0)
          return rows::mul2(e, rows::both(k.A));
        else if constexpr (POW == 2)
          return rows::mul2(e, rows::fma2(e, rows::both(k.B), rows::both(k.A)));
        else
          return rows::fma2(rows::at_one<POW, FAR>(e, q, from1), rows::both(k.B), rows::mul2(e, rows::both(k.A)));
      };
      const bool same_vectors =
          sizeof(TG) == sizeof(TZ)
              ? (reinterpret_cast<uintptr_t>(drow) & 15) / sizeof(TG) == static_cast<uintptr_t>(s.off)
              : s.off == 0 && (reinterpret_cast<uintptr_t>(drow) & (E * sizeof(TG) - 1)) == 0;
      const auto stage = [&](int g, auto far) {
        s.for_stage(sm, g, [&](const uint4& u, int v) {
          float2 q[E / 2];
          rows::to_pairs<TZ>(u, q);
          float out[E];
#pragma unroll
          for (int j = 0; j < E / 2; ++j) {
            const float2 o = gradient(q[j], far);
            out[2 * j] = o.x;
            out[2 * j + 1] = o.y;
          }
          TG* to = drow + s.first + v * E;
          if (same_vectors) {
            store_vec<E>(to, out);
          } else {
#pragma unroll
            for (int j = 0; j < E; ++j) to[j] = from_f32<TG>(out[j]);
          }
        });
      };
#pragma unroll 1
      for (int g = 0; g < kStages; ++g) {
        if (from.far)
          stage(g, std::true_type{});
        else
          stage(g, std::false_type{});
        warp_arrives(&sh.empty[g]);
      }
      if (edge >= 0) {
        const float2 q = rows::both(edge_z);
        drow[edge] = from_f32<TG>((from.far ? gradient(q, std::true_type{}) : gradient(q, std::false_type{})).x);
      }
      if (at.rank == p.parts - 1)
        for (int i = p.vocab + tid; i < p.dz_cols; i += kRingThreads) drow[i] = from_f32<TG>(0.f);
      warp_arrives(&sh.gradient_done[side]);
    }
    on_side ^= 1u << side;
    ++turn;
  }
}

__device__ __forceinline__ float2 warp_sum2(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, v.x, o), b = __shfl_xor_sync(0xffffffffu, v.y, o);
    v.x += a;
    v.y += b;
  }
  return v;
}
// The lanes' sums relative to the largest of their references, which `top` becomes.
template <int POW>
__device__ __forceinline__ float2 relative_sums(float& top, float sum, float sum1, float c) {
  const Ref of(top == -CUDART_INF_F ? 0.f : top, c);
  top = rows::lanes_max(top);
  const Ref to(top == -CUDART_INF_F ? 0.f : top, c);
  const float step = to.log2_of(of, c);
  sum = rows::rescaled(sum, step);
  if (POW != 0)
    sum1 = rows::rescaled(sum1, rows::log2_at_one<POW>(step, rows::ref_at_one<POW>(to), rows::ref_at_one<POW>(of)));
  if (POW == 0) return make_float2(warp_sum(sum), 0.f);
  return warp_sum2(make_float2(sum, sum1));
}

template <typename TG, int FORM, int POW>
__device__ __forceinline__ void finish_rows(TG* dz, Listed* lists, Shared& sh, const Params& p, const Place& at, float c,
                                            float c1) {
  constexpr bool GRAD = FORM != kLoss;
  const int lane = threadIdx.x & 31;
  const float all_scale = scale_of_all(p);
  int turn = 0;
  unsigned on_side = 0;  // bit s: the parity of the live rows side s has had
  for (int n = 0;; ++n) {
    const int side = n % kSides;
    if (!warp_waits(&sh.list_ready[side], (n / kSides) & 1, &sh.stop, p.status)) return;
    const Row& r = sh.row[side];
    if (r.row < 0) return;
    Listed* list = lists + side * p.k;
    // The list's sums, each column once, relative to its largest logit.  With a gradient, whose consumers wait for this
    // warp, already while they sum the last stage (they then cannot run past that stage's phase; without one they can).
    if (!GRAD && !warp_waits(&sh.sums_ready[side], (n / kSides) & 1, &sh.stop, p.status)) return;
    const Ref list_ref(r.list_top, c), list_ref1 = rows::ref_at_one<POW>(list_ref);
    float L = 0.f, L1 = 0.f, listed = 0.f;
    if (r.live) {
      if (GRAD && !warp_waits(&sh.ready[kStages - 1], turn & 1, &sh.stop, p.status)) return;
      const bool repeats = r.repeats;
      const auto add_list = [&] {
        for (int i = lane; i < p.k; i += 32) {
          if (!list[i].owner) continue;
          L += rows::fast_exp2(list_ref.log2_of(list[i].z, c));
          if (POW != 0) L1 += rows::fast_exp2(list_ref1.log2_of(list[i].z, c1));
          listed += 1.f;
        }
      };
      add_list();
      if (__builtin_expect(repeats, 0)) {  // which entry stands for a column decides where it is added: the first, in every run
        for (int i = lane; i < p.k; i += 32)
          if (list[i].stage >= 0) list[i].owner = first_of_column(list, i);
        L = L1 = listed = 0.f;
        add_list();
      }
      L = warp_sum(L);
      if (POW != 0) L1 = warp_sum(L1);
      listed = warp_sum(listed);
    }
    if (GRAD && !warp_waits(&sh.sums_ready[side], (n / kSides) & 1, &sh.stop, p.status)) return;
    if (!r.live) {
      if (FORM != kAgain && lane == 0 && at.rank == 0) p.loss[r.row] = 0.f;
      warp_arrives(&sh.side_free[side]);
      continue;
    }
    const float scale = scale_of<FORM>(p, all_scale, r.row);
    // The unlisted columns' sums, relative to one reference: of this CTA, then of the row.  The consumers wait for what
    // follows, so independent sums go through the lanes together and quotients are the hardware's (2 ulp).
    const rows::WarpSum w = lane < kRingWarps ? sh.sums[side][lane] : rows::WarpSum{-CUDART_INF_F, 0.f, 0.f};
    float rest_top = w.z;
    float2 S2 = relative_sums<POW>(rest_top, w.sum, w.sum1, c);
    if (p.parts > 1) {
      // Two places by turns of live rows: a CTA writes a place again only after the turn between, for which every CTA
      // has arrived after it read this one.
      const Part part{rest_top, S2.x, S2.y, L, L1};
      const int place = turn & 1;
      if (lane < p.parts) {
        *rows::cg::this_cluster().map_shared_rank(&sh.part[place][at.rank], lane) = part;
        mbar_arrive_at(&sh.part_ready[place], lane);
      }
      if (!warp_waits<true>(&sh.part_ready[place], (turn >> 1) & 1, &sh.stop, p.status)) return;
      const Part q = lane < p.parts ? sh.part[place][lane] : Part{-CUDART_INF_F, 0.f, 0.f, 0.f, 0.f};
      rest_top = q.ref;
      S2 = relative_sums<POW>(rest_top, q.sum, q.sum1, c);
      const float2 L2 = warp_sum2(make_float2(q.list, q.list1));
      L = L2.x;
      L1 = L2.y;
    }
    const float S = S2.x, S1 = S2.y;
    const Ref own(rest_top != -CUDART_INF_F ? rest_top : r.list_top, c), own1 = rows::ref_at_one<POW>(own);
    // the row's reference: the larger of the rest's and the list's
    const Ref ref(L != 0.f && r.list_top > own.z ? r.list_top : own.z, c), ref1 = rows::ref_at_one<POW>(ref);
    if (L != 0.f && ref.z != r.list_top) {
      const float step = ref.log2_of(list_ref, c);
      L *= rows::fast_exp2(step);
      if (POW != 0) L1 *= rows::fast_exp2(rows::log2_at_one<POW>(step, ref1, list_ref1));
    }
    const bool same = ref.z == own.z;
    const float step = ref.log2_of(own, c), f = same ? 1.f : rows::fast_exp2(step),
                f1 = same || POW == 0 ? f : rows::fast_exp2(rows::log2_at_one<POW>(step, ref1, own1));
    const float total = S * f + L, total1 = POW != 0 ? S1 * f1 + L1 : total;
    const float inv_sum = __fdividef(1.f, total), inv_sum1 = POW != 0 ? __fdividef(1.f, total1) : inv_sum;
    // a list that names every column leaves no rest, whatever rounding says
    const float m = p.k >= p.vocab && static_cast<int>(listed) >= p.vocab ? 0.f : r.rest;
    const float mass = r.mass + m;
    float A = mass != 0.f ? mass * f * inv_sum : 0.f;
    if (m > 0.f && S > 0.f) A -= __fdividef(m, S);
    A *= scale * p.kd * p.tau;
    float B = p.ce != 0.f ? scale * p.ce * f1 * inv_sum1 : 0.f;
    if (POW == 0) {  // one exponential serves both terms
      A += B;
      B = 0.f;
    }
    if (GRAD) {
      if (lane == 0) sh.scalars[side] = Scalars{own.z, A, B};
      warp_arrives(&sh.scalars_ready[side]);
    }
    const float log2_total = log2f(total);
    float kl = 0.f;
    if (FORM != kAgain && at.rank == 0) {
      for (int i = lane; i < p.k; i += 32) {
        const float logq = (ref.log2_of(list[i].z, c) - log2_total) * CUDART_LN2_F;
        if (list[i].p != 0.f) kl += list[i].p * (list[i].logp - logq);
      }
      kl = warp_sum(kl);
    }
    if (FORM != kAgain && lane == 0 && at.rank == 0) {
      // log q_rest from its parts: the probability itself may leave fp32's range
      if (m > 0.f) kl += m * ((log2f(m) - log2f(S) + log2_total) * CUDART_LN2_F - ref.log_of(own, c, p.inv_tau));
      float loss = p.kd != 0.f ? p.kd * p.tau * p.tau * kl : 0.f;
      if (p.ce != 0.f) loss += p.ce * (log2f(total1) - ref1.log2_of(r.target_logit, c1)) * CUDART_LN2_F;
      p.loss[r.row] = scale * loss;
    }
    if (GRAD) {
      if (!warp_waits(&sh.gradient_done[side], (on_side >> side) & 1, &sh.stop, p.status)) return;
      TG* drow = dz + r.row * p.lddz;
      const float kd = scale * p.kd * p.tau, ce = scale * p.ce;
      for (int i = lane; i < p.k; i += 32) {
        if (!list[i].owner) continue;
        const int col = list[i].col;
        float share = list[i].p;
        if (r.repeats) {
          share = 0.f;
          for (int j = 0; j < p.k; ++j)
            if (list[j].col == col) share += list[j].p;
        }
        float g = kd != 0.f ? kd * (rows::fast_exp2(ref.log2_of(list[i].z, c)) * inv_sum * mass - share) : 0.f;
        if (ce != 0.f) g += ce * (rows::fast_exp2(ref1.log2_of(list[i].z, c1)) * inv_sum1 - (col == r.target ? 1.f : 0.f));
        drow[col] = from_f32<TG>(g);
      }
      if (lane == 0 && ce != 0.f && !r.target_listed && r.target_here) {
        float g = rows::fast_exp2(own.log2_of(r.target_logit, c)) * A - ce;
        if (POW != 0) g += rows::fast_exp2(own1.log2_of(r.target_logit, c1)) * B;
        drow[r.target] = from_f32<TG>(g);
      }
    }
    on_side ^= 1u << side;
    ++turn;
    warp_arrives(&sh.side_free[side]);
  }
}

template <typename TZ, typename TG, int FORM, int POW>
__global__ void __launch_bounds__(kThreads, 2) distill_ring_kernel(const TZ* __restrict__ z, TG* __restrict__ dz,
                                                                  const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  TZ* sm = reinterpret_cast<TZ*>(smem);
  auto* lists = reinterpret_cast<Listed*>(smem + static_cast<size_t>(p.per) * 16);
  if (nothing_to_do<FORM>(p)) return;  // the same for the whole grid
  if (threadIdx.x == 0) {
    for (int g = 0; g < kStages; ++g) {
      mbar_init(&sh.full[g], 1);
      mbar_init(&sh.ready[g], 1);
      mbar_init(&sh.empty[g], kRingWarps);
    }
    for (int i = 0; i < kSides; ++i) {
      mbar_init(&sh.list_ready[i], 1);
      mbar_init(&sh.side_free[i], 2);  // finisher and patcher: the roles that nothing else makes wait for a dead row
      mbar_init(&sh.sums_ready[i], kRingWarps);
      mbar_init(&sh.scalars_ready[i], 1);
      mbar_init(&sh.gradient_done[i], kRingWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&sh.part_ready[i], p.parts);
    sh.stop = 0;
    fence_mbar_init();
  }
  rows::cg::cluster_group cluster = rows::cg::this_cluster();
  if (p.parts > 1)
    cluster.sync();
  else
    __syncthreads();
  const Place at{p.parts > 1 ? static_cast<int>(cluster.block_rank()) : 0, blockIdx.x / p.parts, gridDim.x / p.parts};
  const float c = p.inv_tau * CUDART_L2E_F, c1 = POW == 1 ? CUDART_L2E_F : (POW > 1 ? POW : 1) * c;
  const int warp = threadIdx.x >> 5;
  if (warp < kRingWarps) {
    consume<TZ, TG, FORM, POW>(z, dz, sm, lists, sh, p, at, c);
  } else if (warp == kProducer) {
    if ((threadIdx.x & 31) == 0) produce(z, sm, sh, p, at);
  } else if (warp == kLister) {
    list_rows(z, lists, sh, p, at);
  } else if (warp == kPatcher) {
    patch_stages(sm, lists, sh, p);
  } else {
    finish_rows<TG, FORM, POW>(dz, lists, sh, p, at, c, c1);
  }
  if (p.parts > 1) {  // no CTA leaves while another may still write to it
    __syncwarp();
    cluster.sync();
  }
}

// Clusters of this kernel that the device runs at one time (asked once for each kernel, size and shared memory; an error leaves
// nothing behind).
int active_clusters(const void* kernel, const cudaLaunchConfig_t& cfg, int parts) {
  static std::mutex lock;
  static std::map<std::tuple<int, const void*, int, size_t>, int> known;
  int device = 0;
  TTB_CUDA_CHECK(cudaGetDevice(&device));
  const std::lock_guard<std::mutex> guard(lock);
  const std::tuple<int, const void*, int, size_t> key{device, kernel, parts, cfg.dynamicSmemBytes};
  if (const auto it = known.find(key); it != known.end()) return it->second;
  int clusters = 0;
  TTB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
  return known[key] = clusters < 1 ? 1 : clusters;
}

}  // namespace

bool loss_by_ring(const DistillArgs& a, const Params& params, int pow, cudaStream_t stream) {
  // Shorter rows go a CTA each, several to an SM.  Measured with 8288 rows, 64 listed: 32 KB (16384 bf16) 129 us here and
  // 95 us there, with gradient 176 and 136; 64 KB (32768 bf16) 149 and 195, 232 and 261; (16384 fp32) 127 and 179, 211 and 248.
  constexpr size_t kLeastSlice = 48 * 1024;
  constexpr size_t kMostBytes = 113 * 1024;  // two CTAs on an SM
  const int E = 16 / scalar_bytes(a.z_type);
  const int total = static_cast<int>((a.vocab + 2LL * (E - 1)) / E);  // the most vectors a row can touch
  Params p = params;
  p.rows = a.rows;
  size_t smem = 0;
  for (p.parts = 1; p.parts <= rows::kMaxParts; ++p.parts) {
    p.per = (total + p.parts - 1) / p.parts;
    smem = static_cast<size_t>(p.per) * 16 + kSides * static_cast<size_t>(a.k) * sizeof(Listed);
    if (smem + sizeof(Shared) + 1024 <= kMostBytes) break;
  }
  if (p.parts > rows::kMaxParts || static_cast<size_t>(p.per) * 16 < kLeastSlice || a.rows * p.parts < 4LL * num_sms())
    return false;
  auto launch = [&](auto kernel, auto* z, auto* dz) {
    TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * num_sms());
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    if (p.parts > 1) {
      cfg.gridDim.x = p.parts;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      cfg.gridDim.x = p.parts * active_clusters(reinterpret_cast<const void*>(kernel), cfg, p.parts);
    }
    TTB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, z, dz, p));
  };
  with_kernel_types(a, [&](const auto* z, auto* dz) {
    using TZ = std::remove_const_t<std::remove_pointer_t<decltype(z)>>;
    using TG = std::remove_pointer_t<decltype(dz)>;
    with_pow(pow, [&](auto w) {
      constexpr int POW = decltype(w)::value;
      with_form<TZ, TG>(a, [&](auto form) { launch(distill_ring_kernel<TZ, TG, decltype(form)::value, POW>, z, dz); });
    });
  });
  return true;
}

}  // namespace distill
}  // namespace ttb
