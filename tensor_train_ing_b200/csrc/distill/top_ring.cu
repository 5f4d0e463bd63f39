// A teacher's top logits of many long rows: a persistent kernel whose warps have roles (the method is that of top_logits.cu).
//
//   consumers   stream the rows through a ring of chunks, one after the other without a pause: sums of exponentials and,
//               for every quarter of a row, the largest element of each thread
//   producer    keeps the ring full
//   collectors  behind the consumers: find a bound below the row's k-th largest element from the maxima, read the few
//               threads' vectors that can reach it again (from L2), rank what is found, write it out
//
// No row is kept, so its length does not matter.  8192 rows of 50257 bf16 logits, the top 64, took 264 us with a row per
// CTA (two CTAs of an SM waiting through the bound, the collection and the ranking of each row) and {CHUNK} us here; 2048 rows of
// 131072 fp32 logits, the top 128, {LARGE0} us (a cluster per row) and {LARGE} us.
#include "../common/host.h"
#include "row_ring.cuh"
#include "top_common.cuh"

namespace ttb {
namespace top {
namespace {

using rows::Span;
using rows::kRingThreads;
using rows::kRingWarps;
using rows::wait_for;
using rows::warp_arrives;
using rows::warp_waits;

constexpr int kThreads = 512;
constexpr int kProducer = kRingWarps, kCollector = kRingWarps + 1;
constexpr int kTeam = kThreads - 32 * kCollector;  // collector threads
constexpr int kRounds = 3;                          // vectors of a chunk per consumer thread
constexpr int kChunkVectors = kRounds * kRingThreads;
constexpr int kSlots = 4;
constexpr int kParts = 4;  // a row's quarters
constexpr int kGroups = kParts * kRingThreads;
constexpr int kSides = 3;  // rows between their sums and their end at one time
static_assert(kGroups == 16 * 3 * 32);

struct Shared {
  uint64_t full[kSlots], empty[kSlots];
  uint64_t sums_ready[kSides], side_free[kSides];
  uint32_t maxima[kSides][kGroups];
  rows::WarpSum sums[kSides][kRingWarps];
  unsigned long long list[kCapacity];
  unsigned short hit[kGroups];
  uint32_t bound;
  float total;  // the row's sum relative to top
  float top;
  int hits, taken;
  int red[kTeam / 32], ok[kTeam / 32];
  int stop;
};

template <typename T>
__device__ __forceinline__ int chunks_of(const Span<T>& s) {
  return (s.hi - s.lo + kChunkVectors - 1) / kChunkVectors;
}

template <typename T>
__device__ __forceinline__ void produce(const T* z, long long ldz, long long rows_n, int vocab, T* sm, Shared& sh,
                                        uint32_t* status) {
  unsigned q = 0;
  bool ok = true;
  for (long long row = blockIdx.x; row < rows_n && ok; row += gridDim.x) {
    const Span<T> s(z + row * ldz, vocab, 0, 1 << 30);
    for (int a = s.lo; a < s.hi && ok; a += kChunkVectors, ++q) {
      const unsigned slot = q % kSlots;
      if (q >= kSlots) ok = wait_for(&sh.empty[slot], (q / kSlots - 1) & 1, &sh.stop, status);
      if (!ok) break;
      const int n = min(kChunkVectors, s.hi - a);
      mbar_arrive_expect_tx(&sh.full[slot], n * 16);
      bulk_load(sm + slot * kChunkVectors * Span<T>::kVec, s.row + s.first + a * Span<T>::kVec, n * 16, &sh.full[slot]);
    }
  }
  if (!ok)  // copies under way end before the CTA does
    for (unsigned i = q < kSlots ? 0 : q - kSlots; i < q; ++i)
      mbar_wait(&sh.full[i % kSlots], (i / kSlots) & 1, status, kErrTimeoutProducer);
}

template <typename T>
__device__ __forceinline__ void consume(const T* z, long long ldz, long long rows_n, int vocab, const T* sm, Shared& sh,
                                        float c, uint32_t* status) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned q = 0;
  int n = 0;
  for (long long row = blockIdx.x; row < rows_n; row += gridDim.x, ++n) {
    const int side = n % kSides;
    const Span<T> s(z + row * ldz, vocab, 0, 1 << 30);
    const int edge = tid < 16 ? s.edge_column(tid) : -1;
    const float edge_z = edge >= 0 ? to_f32(s.row[edge]) : 0.f;
    if (n >= kSides && !warp_waits(&sh.side_free[side], (n / kSides - 1) & 1, &sh.stop, status)) return;
    const int chunks = chunks_of(s), each = (chunks + kParts - 1) / kParts;
    rows::Sums<0> sums(c);
    int chunk = 0;
#pragma unroll 1
    for (int part = 0; part < kParts; ++part) {
      float mx = -CUDART_INF_F;
      bool any = false;
#pragma unroll 1
      for (const int end = min(chunks, (part + 1) * each); chunk < end; ++chunk, ++q) {
        const unsigned slot = q % kSlots;
        if (!warp_waits(&sh.full[slot], (q / kSlots) & 1, &sh.stop, status)) return;
        const int have = s.hi - s.lo - chunk * kChunkVectors;
        const T* at = sm + slot * kChunkVectors * Span<T>::kVec;
#pragma unroll 1
        for (int i = tid; i < min(have, kChunkVectors); i += kRingThreads) {
          const uint4 u[1] = {*reinterpret_cast<const uint4*>(at + i * Span<T>::kVec)};
          const float top = rows::max_of<T>(u);
          mx = fmaxf(mx, top);
          any = true;
          sums.see(top, c);
          sums.template add_batch<T>(u, c);
        }
        warp_arrives(&sh.empty[slot]);
      }
      sh.maxima[side][part * kRingThreads + tid] = any ? ordered(mx) : 0u;
    }
    if (edge >= 0) sums.add_one(edge_z, c);
    const rows::WarpSum mine = rows::warp_total<0>(sums, c, c);
    if (lane == 0) sh.sums[side][warp] = mine;
    warp_arrives(&sh.sums_ready[side]);
  }
}

__device__ __forceinline__ void team_barrier() { named_barrier(1, kTeam); }

__device__ __forceinline__ int team_count(int v, int* red, int warp) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  team_barrier();
  int t = 0;
#pragma unroll
  for (int i = 0; i < kTeam / 32; ++i) t += red[i];
  team_barrier();
  return t;
}

template <typename T>
__device__ __forceinline__ void collect(const T* z, long long ldz, long long rows_n, int vocab, int k, float inv_tau,
                                        T* values, int* ids, float* lse, Shared& sh, float c, uint32_t* status) {
  constexpr int E = Span<T>::kVec;
  const int t = threadIdx.x - 32 * kCollector, lane = t & 31, warp = t >> 5;
  const auto take = [&](float value, int col) {
    const int to = atomicAdd(&sh.taken, 1);
    if (to < kCapacity) sh.list[to] = key_of(value, col);
  };
  int n = 0;
  for (long long row = blockIdx.x; row < rows_n; row += gridDim.x, ++n) {
    const int side = n % kSides;
    const bool ok = warp_waits(&sh.sums_ready[side], (n / kSides) & 1, &sh.stop, status);
    if (lane == 0) sh.ok[warp] = ok;
    if (t == 0) sh.hits = sh.taken = 0;
    team_barrier();
    bool all_ok = true;
#pragma unroll
    for (int i = 0; i < kTeam / 32; ++i) all_ok &= sh.ok[i] != 0;
    if (!all_ok) return;  // the whole team: none is left at its barrier
    const Span<T> s(z + row * ldz, vocab, 0, 1 << 30);
    if (warp == 0) {
      const uint32_t bound = find_bound<T, 3>(sh.maxima[side], kGroups, k);
      if (lane == 0) sh.bound = bound;
    } else if (warp == 1) {
      const rows::WarpSum w = lane < kRingWarps ? sh.sums[side][lane] : rows::WarpSum{-CUDART_INF_F, 0.f, 0.f};
      const float top = warp_max(w.z);
      const rows::Ref ref(top == -CUDART_INF_F ? 0.f : top, c), of(w.z == -CUDART_INF_F ? 0.f : w.z, c);
      const float total = warp_sum(rows::rescaled(w.sum, ref.log2_of(of, c)));
      if (lane == 0) {
        sh.total = total;
        sh.top = ref.z;
        lse[row] = ref.far ? ref.z * inv_tau + logf(total) : (ref.r + log2f(total)) * CUDART_LN2_F;
      }
    }
    team_barrier();
    const uint32_t bound = sh.bound;
    // NaN, or no bound: the k-th largest element is searched bit by bit
    bool search = sh.total != sh.total || bound <= ordered(-CUDART_INF_F);
    if (!search) {
      const float least = from_ordered(bound);
      for (int g = t; g < kGroups; g += kTeam) {
        const bool hit = sh.maxima[side][g] >= bound;
        const unsigned who = __ballot_sync(0xffffffffu, hit);
        if (who == 0) continue;
        int at = 0;
        if (lane == 0) at = atomicAdd(&sh.hits, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0);
        if (hit) sh.hit[at + __popc(who & ((1u << lane) - 1u))] = static_cast<unsigned short>(g);
      }
      const int edge = t < 16 ? s.edge_column(t) : -1;
      if (edge >= 0) {
        const float v = to_f32(s.row[edge]);
        if (v >= least) take(v, edge);
      }
      team_barrier();
      // `lanes` threads look through a group's vectors, two groups at a time so that their reads overlap
      const int chunks = chunks_of(s), each = (chunks + kParts - 1) / kParts, rounds = each * kRounds;
      const int lanes = rounds <= 8 ? 8 : rounds <= 16 ? 16 : 32, teams = kTeam / lanes;
      const int hits = sh.hits, in = t % lanes;
      for (int h = t / lanes; h < hits; h += 2 * teams) {
        for (int j = in; j < rounds; j += lanes) {
          uint4 u[2];
          int first[2];
          bool have[2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int hit = h + b * teams;
            const int g = hit < hits ? sh.hit[hit] : 0, part = g / kRingThreads, who = g % kRingThreads;
            const int v = s.lo + (part * rounds + j) * kRingThreads + who;
            have[b] = hit < hits && v < s.hi;
            first[b] = s.first + v * E;
            if (have[b]) u[b] = __ldg(reinterpret_cast<const uint4*>(s.row + first[b]));
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (!have[b]) continue;
            float2 q[E / 2];
            rows::to_pairs<T>(u[b], q);
#pragma unroll
            for (int e = 0; e < E / 2; ++e) {
              if (q[e].x >= least) take(q[e].x, first[b] + 2 * e);
              if (q[e].y >= least) take(q[e].y, first[b] + 2 * e + 1);
            }
          }
        }
      }
      team_barrier();
      search = sh.taken > kCapacity;
    }
    int total = sh.taken;
    if (search) {
      const int col_bits = 32 - __clz(vocab);  // the column's upper bits are ones in every key
      unsigned long long kth = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long trial = kth | (1ull << bit);
        if (bit < 32 && bit >= col_bits) {
          kth = trial;
          continue;
        }
        int m = 0;
        for (int col = t; col < vocab; col += kTeam) m += key_of(to_f32(s.row[col]), col) >= trial;
        if (team_count(m, sh.red, warp) >= k) kth = trial;
      }
      if (t == 0) sh.taken = 0;
      team_barrier();
      for (int col = t; col < vocab; col += kTeam) {
        const float v = to_f32(s.row[col]);
        if (key_of(v, col) >= kth) take(v, col);
      }
      team_barrier();
      total = k;
    }
    for (int i = t; i < total; i += kTeam) {
      const unsigned long long key = sh.list[i];
      int place = 0;
      for (int j = 0; j < total; ++j) place += sh.list[j] > key;
      if (place < k) {
        values[row * k + place] = from_f32<T>(from_ordered(static_cast<uint32_t>(key >> 32)));
        ids[row * k + place] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
      }
    }
    team_barrier();  // the list and the counters may be used again
    if (t == 0) mbar_arrive(&sh.side_free[side]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) top_ring_kernel(const T* __restrict__ z, long long ldz, long long rows_n,
                                                              int vocab, int k, float inv_tau, T* __restrict__ values,
                                                              int* __restrict__ ids, float* __restrict__ lse,
                                                              uint32_t* status) {
  extern __shared__ __align__(16) uint8_t smem[];
  T* sm = reinterpret_cast<T*>(smem);
  Shared& sh = *reinterpret_cast<Shared*>(smem + kSlots * kChunkVectors * 16);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], kRingWarps);
    }
    for (int i = 0; i < kSides; ++i) {
      mbar_init(&sh.sums_ready[i], kRingWarps);
      mbar_init(&sh.side_free[i], 1);
    }
    sh.stop = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const float c = inv_tau * CUDART_L2E_F;
  const int warp = threadIdx.x >> 5;
  if (warp < kRingWarps) {
    consume(z, ldz, rows_n, vocab, sm, sh, c, status);
  } else if (warp == kProducer) {
    if ((threadIdx.x & 31) == 0) produce(z, ldz, rows_n, vocab, sm, sh, status);
  } else {
    collect(z, ldz, rows_n, vocab, k, inv_tau, values, ids, lse, sh, c, status);
  }
}

}  // namespace

bool top_logits_by_ring(const TopLogitsArgs& a, cudaStream_t stream) {
  const long long bytes = static_cast<long long>(a.vocab) * scalar_bytes(a.type);
  // Shorter rows leave the collectors less time than they need; few rows leave CTAs without any.
  if (bytes < 32 * 1024 || a.rows < 4LL * num_sms()) return false;
  const size_t smem = kSlots * kChunkVectors * 16 + sizeof(Shared);
  with_type(a.type, [&](auto* tz) {
    using T = std::remove_pointer_t<decltype(tz)>;
    auto kernel = top_ring_kernel<T>;
    TTB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    kernel<<<2 * num_sms(), kThreads, smem, stream>>>(static_cast<const T*>(a.z), a.ldz, a.rows, a.vocab, a.k,
                                                      a.inv_tau, static_cast<T*>(a.values), a.ids, a.lse,
                                                      status_ptr());
  });
  TTB_CUDA_CHECK(cudaGetLastError());
  return true;
}

}  // namespace top
}  // namespace ttb
