// The token that a thread of a cache write takes: plain arithmetic, for host and device.
#pragma once

#include <cstdint>

#ifndef __HIPCC__
#define __host__
#define __device__
#endif

namespace paged {

// Token of row `row` of workgroup `group`, `rows` tokens to each; -1 past the last.  (In 64
// bits: one grid serves walks of different `rows`, and the one of more tokens a workgroup
// has workgroups that start past 2^31.)
__host__ __device__ constexpr int32_t token_of(uint32_t group, int32_t rows, int32_t row,
                                               int32_t tokens) {
  const int64_t token = (int64_t)group * rows + row;
  return row < rows && token < tokens ? (int32_t)token : -1;
}

}  // namespace paged
