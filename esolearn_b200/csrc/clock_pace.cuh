// Pacing by the SM's clock counter.  No CUDA in here, so that the host can test it.
#pragma once

#include <cstdint>

namespace sb {

// Whether `now` lies n clocks or more behind `from`, both read from the 32-bit
// counter, which wraps about every two seconds: their difference modulo 2^32 is
// the number of clocks between them, wherever the wrap falls.
constexpr bool clocks_passed(uint32_t from, uint32_t now, uint32_t n) { return now - from >= n; }

}  // namespace sb
