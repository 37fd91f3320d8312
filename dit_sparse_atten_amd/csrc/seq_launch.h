// Launches of the sequence attention kernels of one element type.
#pragma once

#include <algorithm>

#include "seq_attn.h"

namespace seq {

template <typename T, int kD, int kUse>
void launch_wide(const Params& p, bool paged, dim3 grid, hipStream_t stream) {
  if (paged) hipLaunchKernelGGL((seq_wide_kernel<T, kD, kUse, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((seq_wide_kernel<T, kD, kUse, false>), grid, dim3(256), 0, stream, p);
}

// The join of split tiles.
template <typename T, int kD>
void launch_merge(const Params& p, bool narrow, hipStream_t stream) {
  const int units = (narrow ? kNarrowRows : kWideRows) / 16;
  // Tiles have many parts only where there are few of them.
  const bool few_tiles = (int64_t)p.max_tiles * kFewParts <= p.max_slots;
  const dim3 groups((unsigned)std::min<int64_t>((int64_t)p.max_splits * units,
                                                std::max(1, 2048 / p.kv_heads)),
                    (unsigned)p.kv_heads, few_tiles ? 16u : 1u);
  const dim3 block(256);
  if (narrow) hipLaunchKernelGGL((seq_merge_kernel<T, kD, kNarrowRows>), groups, block, 0, stream, p);
  else hipLaunchKernelGGL((seq_merge_kernel<T, kD, kWideRows>), groups, block, 0, stream, p);
}

template <typename T, int kD>
int launch_dim(const Params& p, bool paged, bool narrow, int max_groups, bool merge,
               hipStream_t stream, const char* who) {
  const dim3 grid((unsigned)max_groups), narrow_block(kNarrowWaves * 64);
  if (narrow) {
    if (paged) hipLaunchKernelGGL((seq_narrow_kernel<T, kD, true>), grid, narrow_block, 0, stream, p);
    else hipLaunchKernelGGL((seq_narrow_kernel<T, kD, false>), grid, narrow_block, 0, stream, p);
  } else if (kD == 128 && p.head_dim <= 96) {
    launch_wide<T, kD, kD == 128 ? 96 : kD>(p, paged, grid, stream);
  } else {
    launch_wide<T, kD, kD>(p, paged, grid, stream);
  }
  if (merge) launch_merge<T, kD>(p, narrow, stream);
  return dsa::check_launch(who);
}

template <typename T>
int launch_typed(const Params& p, bool paged, bool narrow, int max_groups, bool merge,
                 hipStream_t stream, const char* who) {
  return p.head_dim <= 64
             ? launch_dim<T, 64>(p, paged, narrow, max_groups, merge, stream, who)
             : launch_dim<T, 128>(p, paged, narrow, max_groups, merge, stream, who);
}

}  // namespace seq
