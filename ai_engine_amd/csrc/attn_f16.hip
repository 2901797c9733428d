// attn_f16.hip -- the f16 instances of the attention kernel (attn_impl.h).
#include "attn_impl.h"

namespace aih {

hipError_t launch_attn_f16(const AttnArgs &a, int kernel, hipStream_t st) {
  return at_launch_dt<DT_F16>(a, kernel, st);
}

}  // namespace aih
