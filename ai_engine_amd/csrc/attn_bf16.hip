// attn_bf16.hip -- the bf16 instances of the attention kernel (attn_impl.h).
#include "attn_impl.h"

namespace aih {

hipError_t launch_attn_bf16(const AttnArgs &a, int kernel, hipStream_t st) {
  return at_launch_dt<DT_BF16>(a, kernel, st);
}

}  // namespace aih
