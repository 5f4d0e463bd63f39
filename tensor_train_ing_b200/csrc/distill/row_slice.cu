#include "row_slice.cuh"

#include "../common/host.h"
#include "distill_api.h"

namespace ttb {
namespace rows {

Plan plan_rows(long long rows, int cols, int elem_bytes) {
  const int E = 16 / elem_bytes;
  const int total = (cols + 2 * (E - 1)) / E;  // the most vectors a row can touch
  Plan p;
  p.parts = 1;
  while (p.parts < kMaxParts && static_cast<size_t>((total + p.parts - 1) / p.parts) * 16 > 32 * 1024) p.parts *= 2;
  while (p.parts < kMaxParts && rows * p.parts < num_sms() && total / p.parts > 256) p.parts *= 2;
  p.per = (total + p.parts - 1) / p.parts;
  p.threads = 256;
  p.slice_bytes = static_cast<size_t>(p.per) * 16;
  return p;
}

}  // namespace rows

bool logits_row_fits(int cols, ScalarType type) {
  const int E = 16 / scalar_bytes(type);
  const long long total = (cols + 2LL * (E - 1)) / E;
  return (total + rows::kMaxParts - 1) / rows::kMaxParts * 16 <= static_cast<long long>(rows::kMaxSliceBytes);
}

}  // namespace ttb
