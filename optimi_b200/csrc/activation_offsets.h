// Which calls of the activation kernels may compute their offsets in 32 bits.  Plain C++: a host compiler takes it too.
#pragma once
#include <cstdint>

namespace optimi {
namespace act {

// Whether the offsets into `rows` rows of values, of codes and of exponents (`stride`, `pitch` and `epitch` elements apart), and those
// of the items a last block reaches past the end, fit 32 bits.  rows: 1 or more; the others: 0 or more.
constexpr bool small_offsets(int64_t rows, int64_t stride, int64_t pitch, int64_t epitch) {
  const int64_t most = ((1ll << 31) - (1 << 20)) / rows;
  return stride < most && pitch < most && epitch < most;
}

}  // namespace act
}  // namespace optimi
