// fp16 instances of the packed and paged sequence attention (seq_attn.h).
#include "seq_launch.h"

int seq_launch_f16(const seq::Params& p, bool paged, bool narrow, int max_groups, bool merge,
                   hipStream_t stream, const char* who) {
  return seq::launch_typed<_Float16>(p, paged, narrow, max_groups, merge, stream, who);
}
