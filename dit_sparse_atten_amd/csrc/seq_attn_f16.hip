// fp16 instances of the packed and paged sequence attention (seq_attn.h).
#include "seq_launch.h"

int seq_launch_f16(const seq::Params& p, bool paged, bool narrow, int max_groups, bool merge,
                   hipStream_t stream, const char* who) {
  return seq::launch_typed<_Float16>(p, paged, narrow, max_groups, merge, stream, who);
}

void seq_merge_f16(const seq::Params& p, bool narrow, hipStream_t stream) {
  if (p.head_dim <= 64) seq::launch_merge<_Float16, 64>(p, narrow, stream);
  else seq::launch_merge<_Float16, 128>(p, narrow, stream);
}
