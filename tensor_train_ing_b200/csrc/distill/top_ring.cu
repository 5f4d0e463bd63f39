// A teacher's top logits of many long rows: a persistent kernel whose warps have roles (the method is that of top_logits.cu).
//
//   consumers   stream the rows through a ring of chunks, one after the other without a pause: sums of exponentials and,
//               for every quarter of a row and each thread, the largest element, the vector that has it, and the largest
//               element of the thread's other vectors
//   producer    keeps the ring full
//   collectors  behind the consumers, a row each: find a bound below the row's k-th largest element from the maxima, read
//               the vectors that can reach it again (from L2; one of a thread, mostly), rank what is found, write it
//
// No row is kept, so its length does not matter.  8192 rows of 50257 bf16 logits, the top 64, took 264 us with a row per
// CTA (two CTAs of an SM waiting through the bound, the collection and the ranking of each row) and 236 us here (126 us for
// the bytes).  No unit is full (issue slots 62 %, special functions 40 %, DRAM 42 %): the consumers' chain of load, maximum, leaders
// and exponentials of one vector waits for itself.  2048 rows of 131072 fp32 logits, the top 128, took 515 us with a
// cluster per row and 204 us here (165 us).  Rows with fewer than k logits above -inf, and rows with NaN, are searched by a
// collector alone: 2048 rows of 131072 with 200 such logits took 86 ms for the top 128.
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
constexpr int kCollectors = kThreads / 32 - kCollector;
constexpr int kRounds = 4;                          // vectors of a chunk per consumer thread
constexpr int kChunkVectors = kRounds * kRingThreads;
constexpr int kSlots = 2;
constexpr int kParts = 4;  // a row's quarters
constexpr int kGroups = kParts * kRingThreads;
constexpr int kSides = 3;  // rows between their sums and their end at one time
static_assert(kGroups == 16 * 3 * 32);
constexpr int kMostHits = 640;  // groups at the bound that are looked through; more (ties) are searched

struct Shared {
  uint64_t full[kSlots], empty[kSlots];
  uint64_t sums_ready[kSides], side_free[kSides];
  uint32_t maxima[kSides][kGroups];
  uint32_t others[kSides][kGroups];  // upper 16 bits of ordered(next) above the vector's number
  rows::WarpSum sums[kSides][kRingWarps];
  unsigned long long list[kCollectors][kCapacity];
  uint32_t hit[kCollectors][kMostHits];
  int taken[kCollectors];
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
    const float edge_z = edge >= 0 ? to_f32(rows::load_early(s.row + edge)) : 0.f;
    if (n >= kSides && !warp_waits(&sh.side_free[side], (n / kSides - 1) & 1, &sh.stop, status)) return;
    const int chunks = chunks_of(s), each = (chunks + kParts - 1) / kParts;
    rows::Sums<0> sums(c);
    bool sure = false;  // all threads of the warp have a reference: vectors are added without looking for one
    int chunk = 0;
#pragma unroll 1
    for (int part = 0; part < kParts; ++part) {
      rows::Leaders lead;
      int number = 0;
      const bool any = s.lo + part * each * kChunkVectors + tid < s.hi;
#pragma unroll 1
      for (const int end = min(chunks, (part + 1) * each); chunk < end; ++chunk, ++q) {
        const unsigned slot = q % kSlots;
        if (!warp_waits(&sh.full[slot], (q / kSlots) & 1, &sh.stop, status)) return;
        const int have = min(s.hi - s.lo - chunk * kChunkVectors, kChunkVectors);
        const T* at = sm + slot * kChunkVectors * Span<T>::kVec;
        if (sure) {
#pragma unroll 1
          for (int i = tid; i < have; i += kRingThreads) {
            const uint4 u = *reinterpret_cast<const uint4*>(at + i * Span<T>::kVec);
            lead.take(rows::max_of<T>(u), number++);
            sums.template add_vector<T, false>(u, c);
          }
        } else {
#pragma unroll 1
          for (int i = tid; i < have; i += kRingThreads) {
            const uint4 u = *reinterpret_cast<const uint4*>(at + i * Span<T>::kVec);
            const float top = rows::max_of<T>(u);
            lead.take(top, number++);
            sums.see(top, c);
            sums.template add_seen<T>(u, c);
          }
          sure = sums.settle(c);
        }
        warp_arrives(&sh.empty[slot]);
      }
      sh.maxima[side][part * kRingThreads + tid] = any ? ordered(lead.most) : 0u;
      sh.others[side][part * kRingThreads + tid] = (ordered(lead.next) & 0xFFFF0000u) | static_cast<uint32_t>(lead.where);
    }
    if (edge >= 0) sums.add_one(edge_z, c);
    if (sums.overflowed()) {  // rare: logits 40 tau above a thread's first ones, infinities, NaN
      sums = rows::Sums<0>(c);
      for (int v = s.lo + tid; v < s.hi; v += kRingThreads)
        for (int e = 0; e < Span<T>::kVec; ++e) sums.add_one(to_f32(s.row[s.first + v * Span<T>::kVec + e]), c);
      if (edge >= 0) sums.add_one(edge_z, c);
    }
    const rows::WarpSum mine = rows::warp_total<0>(sums, c);
    if (lane == 0) sh.sums[side][warp] = mine;
    warp_arrives(&sh.sums_ready[side]);
  }
}

// f(element, column) over a row, by one warp.
template <typename T, typename F>
__device__ __forceinline__ void each_element(const Span<T>& s, int lane, F&& f) {
  constexpr int E = Span<T>::kVec;
#pragma unroll 2
  for (int v = s.lo + lane; v < s.hi; v += 32) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(s.row + s.first + v * E));
    float2 q[E / 2];
    rows::to_pairs<T>(u, q);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      f(q[e].x, s.first + v * E + 2 * e);
      f(q[e].y, s.first + v * E + 2 * e + 1);
    }
  }
  const int edge = lane < 16 ? s.edge_column(lane) : -1;
  if (edge >= 0) f(to_f32(s.row[edge]), edge);
}

__device__ __forceinline__ void put(unsigned long long* list, int* taken, unsigned long long key) {
  const int to = atomicAdd(taken, 1);
  if (to < kCapacity) list[to] = key;
}

// One warp: the k largest keys of a row into the list, by finding the k-th bit by bit.  Out of line: it is rare, and its
// registers and code should not weigh on the usual way.
template <typename T>
__device__ __noinline__ void search_row(const Span<T>& s, int vocab, int k, unsigned long long* list, int* taken) {
  const int lane = threadIdx.x & 31;
  const int col_bits = 32 - __clz(vocab);  // the column's upper bits are ones in every key
  unsigned long long kth = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long trial = kth | (1ull << bit);
    if (bit < 32 && bit >= col_bits) {
      kth = trial;
      continue;
    }
    int m = 0;
    each_element<T>(s, lane, [&](float v, int col) { m += key_of(v, col) >= trial; });
    if (__reduce_add_sync(0xffffffffu, m) >= k) kth = trial;
  }
  if (lane == 0) *taken = 0;
  __syncwarp();
  each_element<T>(s, lane, [&](float v, int col) {
    if (key_of(v, col) >= kth) put(list, taken, key_of(v, col));
  });
  __syncwarp();
}

// Writes those of the keys first, first + 1, ... (M per lane) that are among the k largest of all to their places.
template <int M, typename T>
__device__ __forceinline__ void rank(const unsigned long long* list, int total, int k, T* values, int* ids,
                                     int first = 0) {
  const int lane = threadIdx.x & 31;
  unsigned long long key[M];
  int place[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int i = first + lane + 32 * m;
    key[m] = i < total ? list[i] : 0ull;
    place[m] = i < total ? 0 : k;
  }
#pragma unroll 2
  for (int j = 0; j < total; ++j) {
    const unsigned long long other = list[j];
#pragma unroll
    for (int m = 0; m < M; ++m) place[m] += other > key[m];
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
    if (place[m] >= k) continue;
    values[place[m]] = from_f32<T>(from_ordered(static_cast<uint32_t>(key[m] >> 32)));
    ids[place[m]] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key[m]));
  }
}

template <typename T>
__device__ __forceinline__ void collect(const T* z, long long ldz, long long rows_n, int vocab, int k, float inv_tau,
                                        T* values, int* ids, float* lse, Shared& sh, float c, uint32_t* status) {
  constexpr int E = Span<T>::kVec;
  const int lane = threadIdx.x & 31, me = (threadIdx.x >> 5) - kCollector;
  unsigned long long* list = sh.list[me];
  uint32_t* hit_list = sh.hit[me];
  int& taken = sh.taken[me];
  const auto take = [&](float value, int col) {
    put(list, &taken, key_of(value, col));
  };
  int n = me;
  for (long long row = blockIdx.x + static_cast<long long>(me) * gridDim.x; row < rows_n;
       row += static_cast<long long>(kCollectors) * gridDim.x, n += kCollectors) {
    const int side = n % kSides;
    if (!warp_waits(&sh.sums_ready[side], (n / kSides) & 1, &sh.stop, status)) return;
    if (lane == 0) taken = 0;
    __syncwarp();
    const Span<T> s(z + row * ldz, vocab, 0, 1 << 30);
    const rows::WarpSum w = lane < kRingWarps ? sh.sums[side][lane] : rows::WarpSum{-CUDART_INF_F, 0.f, 0.f};
    const float top = warp_max(w.z);
    const rows::Ref ref(top == -CUDART_INF_F ? 0.f : top, c), of(w.z == -CUDART_INF_F ? 0.f : w.z, c);
    const float sum = warp_sum(rows::rescaled(w.sum, ref.log2_of(of, c)));
    if (lane == 0) lse[row] = ref.far ? ref.z * inv_tau + logf(sum) : (ref.r + log2f(sum)) * CUDART_LN2_F;
    // three groups as one, unless k is more than a quarter of what is left then
    const uint32_t bound =
        k <= kGroups / 12 ? find_bound<T, 3>(sh.maxima[side], kGroups, k) : find_close_bound<T>(sh.maxima[side], kGroups, k);
    // Groups that can hold elements at the bound: those in which only one vector can from the list's front, the others from its
    // end.  Then the side's maxima are free.
    const float least = from_ordered(bound);
    // NaN, no bound, or too many groups at it: the k-th largest element is searched bit by bit
    bool search = sum != sum || bound <= ordered(-CUDART_INF_F);
    int one = 0, several = 0;
    for (int g = lane; g < kGroups && !search; g += 32) {
      const bool hit = sh.maxima[side][g] >= bound;
      if (!__any_sync(0xffffffffu, hit)) continue;
      const uint32_t other = sh.others[side][g];
      const bool more = hit && (other | 0xFFFFu) >= bound;
      const unsigned singles = __ballot_sync(0xffffffffu, hit && !more), multis = __ballot_sync(0xffffffffu, more);
      const unsigned below = (1u << lane) - 1u;
      const int to = more ? kMostHits - 1 - several - __popc(multis & below) : one + __popc(singles & below);
      one += __popc(singles);
      several += __popc(multis);
      search = one + several > kMostHits;
      if (hit && !search) hit_list[to] = static_cast<uint32_t>(g) << 16 | (other & 0xFFFFu);
    }
    warp_arrives(&sh.side_free[side]);
    if (!search) {
      const int edge = lane < 16 ? s.edge_column(lane) : -1;
      if (edge >= 0) {
        const float v = to_f32(s.row[edge]);
        if (v >= least) take(v, edge);
      }
      constexpr int U = 4;  // vectors a lane reads at a time
      const int chunks = chunks_of(s), each = (chunks + kParts - 1) / kParts, rounds = each * kRounds;
      const auto column = [&](uint32_t hit, int round) {  // of the vector in this round of the group
        const int g = static_cast<int>(hit >> 16), part = g / kRingThreads;
        return s.first + (s.lo + (part * rounds + round) * kRingThreads + g % kRingThreads) * E;
      };
      const auto look = [&](const uint4 (&u)[U], const int (&first)[U], const bool (&have)[U]) {
#pragma unroll
        for (int b = 0; b < U; ++b) {
          if (!have[b]) continue;
          float2 q[E / 2];
          rows::to_pairs<T>(u[b], q);
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            if (q[e].x >= least) take(q[e].x, first[b] + 2 * e);
            if (q[e].y >= least) take(q[e].y, first[b] + 2 * e + 1);
          }
        }
      };
      for (int h = lane; h < one; h += 32 * U) {
        uint4 u[U];
        int first[U];
        bool have[U];
#pragma unroll
        for (int b = 0; b < U; ++b) {
          have[b] = h + 32 * b < one;
          const uint32_t hit = have[b] ? hit_list[h + 32 * b] : 0u;
          first[b] = column(hit, hit & 0xFFFFu);
          if (have[b]) u[b] = __ldg(reinterpret_cast<const uint4*>(s.row + first[b]));
        }
        look(u, first, have);
      }
      // `lanes` lanes look through all vectors of a group, four groups at a time so that their reads overlap
      const int lanes = rounds <= 8 ? 8 : rounds <= 16 ? 16 : 32, teams = 32 / lanes;
      for (int h = lane / lanes; h < several; h += U * teams) {
        for (int j = lane % lanes; j < rounds; j += lanes) {
          uint4 u[U];
          int first[U];
          bool have[U];
#pragma unroll
          for (int b = 0; b < U; ++b) {
            const int hit = h + b * teams;
            first[b] = hit < several ? column(hit_list[kMostHits - 1 - hit], j) : 0;
            have[b] = hit < several && first[b] < s.first + s.hi * E;
            if (have[b]) u[b] = __ldg(reinterpret_cast<const uint4*>(s.row + first[b]));
          }
          look(u, first, have);
        }
      }
      __syncwarp();
      search = taken > kCapacity;
    }
    int total = taken;
    __syncwarp();
    if (search) {
      search_row<T>(s, vocab, k, list, &taken);
      total = k;
    }
    if (total <= 96)
      rank<3>(list, total, k, values + row * k, ids + row * k);
    else
      for (int first = 0; first < total; first += 256) rank<8>(list, total, k, values + row * k, ids + row * k, first);
    __syncwarp();  // the list is filled again
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
  if (bytes / 16 / kRingThreads > 0xFFFF) return false;  // a vector's number is kept in 16 bits
  // A collector's time per row grows with k, a consumer's with the row's length.  Measured with 8288 bf16 rows, here and
  // with a row per CTA: 32768 columns, top 8 150 and 149 us, top 64 216 and 182; 40960 columns 165 and 210, 220 and 247,
  // top 128 349 and 317.  4144 fp32 rows of 32768 columns: top 8 100 and 192 us, top 128 173 and 259.
  if (bytes < 80 * 1024 || a.k * 1024LL > bytes) return false;
  if (a.rows < 4LL * num_sms()) return false;  // few rows leave CTAs without any
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
