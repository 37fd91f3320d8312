// Attention over a paged cache of 4-bit elements: launches of seq_attn_fp4.h's kernels.
#include "seq_attn_fp4.h"

#include "seq_launch.h"

namespace seq {

template <typename T, int kD>
void launch_fp4(const Params& p, bool narrow, dim3 grid, hipStream_t stream) {
  if (narrow && p.slots == kFp4Slots)
    hipLaunchKernelGGL((seq_narrow_fp4_kernel<T, kD, 4>), grid, dim3(256), 0, stream, p);
  else if (narrow)
    hipLaunchKernelGGL((seq_narrow_fp4_kernel<T, kD, 8>), grid, dim3(512), 0, stream, p);
  else if (kD == 128 && p.head_dim <= 96)
    hipLaunchKernelGGL((seq_wide_fp4_kernel<T, kD, kD == 128 ? 96 : kD>), grid, dim3(256), 0,
                       stream, p);
  else
    hipLaunchKernelGGL((seq_wide_fp4_kernel<T, kD, kD>), grid, dim3(256), 0, stream, p);
}

}  // namespace seq

int seq_launch_fp4(const seq::Params& p, int32_t dtype, bool narrow, int max_groups, bool merge,
                   hipStream_t stream, const char* who) {
  const dim3 grid((unsigned)max_groups);
  if (dtype == DSA_BF16) {
    if (p.head_dim <= 64) seq::launch_fp4<__bf16, 64>(p, narrow, grid, stream);
    else seq::launch_fp4<__bf16, 128>(p, narrow, grid, stream);
  } else {
    if (p.head_dim <= 64) seq::launch_fp4<_Float16, 64>(p, narrow, grid, stream);
    else seq::launch_fp4<_Float16, 128>(p, narrow, grid, stream);
  }
  if (merge) dtype == DSA_BF16 ? seq_merge_bf16(p, narrow, stream) : seq_merge_f16(p, narrow, stream);
  return dsa::check_launch(who);
}
