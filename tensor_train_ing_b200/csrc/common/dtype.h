// Element types of the operators that take fp32, bf16 and fp16 rows.
#pragma once

namespace ttb {

enum class ScalarType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

inline int scalar_bytes(ScalarType t) { return t == ScalarType::kF32 ? 4 : 2; }

}  // namespace ttb
