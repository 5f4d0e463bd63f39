#include "row_slice.cuh"

#include "../common/host.h"
#include "distill_api.h"

namespace ttb {
namespace rows {

namespace {
// Two slices of this size and their lists fit an SM: one row's copies run under the other's arithmetic.
constexpr size_t kTargetSliceBytes = 104 * 1024;
}  // namespace

Plan plan_rows(long long rows, int cols, int elem_bytes) {
  const int E = 16 / elem_bytes;
  const int total = (cols + 2 * (E - 1)) / E;  // the most vectors a row can touch
  auto slice = [&](int parts) { return static_cast<size_t>((total + parts - 1) / parts) * 16; };
  Plan p;
  p.parts = 1;
  while (p.parts < kMaxParts && slice(p.parts) > kTargetSliceBytes) p.parts *= 2;
  while (p.parts < kMaxParts && rows * p.parts < num_sms() && total / p.parts > 512) p.parts *= 2;
  p.per = (total + p.parts - 1) / p.parts;
  p.slice_bytes = slice(p.parts);
  // Many rows: about 8 to 16 vectors per thread, so that what every warp does once per row weighs little.  Few rows:
  // more threads, for the latency of one row.
  const int most = rows * p.parts < 2 * num_sms() ? 4 : 16;
  p.threads = 128;
  while (p.threads < kMaxThreads && p.per > p.threads * most) p.threads *= 2;
  return p;
}

}  // namespace rows

bool logits_row_fits(int cols, ScalarType type) {
  const int E = 16 / scalar_bytes(type);
  const long long total = (cols + 2LL * (E - 1)) / E;
  return (total + rows::kMaxParts - 1) / rows::kMaxParts * 16 <= static_cast<long long>(rows::kMaxSliceBytes);
}

}  // namespace ttb
