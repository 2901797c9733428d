// kv4_attn_bf16.hip -- the bf16 instances of the attention over a 4-bit cache.
#include "kv4_attn_impl.h"

namespace aih {

hipError_t launch_kv4_attn_bf16(const Kv4AttnArgs &a, hipStream_t st) { return kv_launch_dt<DT_BF16>(a, st); }

}  // namespace aih
