// attn_f16.hip -- the f16 instances of the attention kernels.
#include "attn_keys.h"
#include "attn_rows.h"

namespace aih {

hipError_t launch_attn_f16(const AttnArgs &a, int kernel, hipStream_t st) {
  const uint32_t cus = device_cus();
#define AIH_AT_CASE(DP)                                                                   \
  if (a.d <= DP) {                                                                        \
    if constexpr (kAtRowsFit<DT_F16, DP>)                                                 \
      if (kernel == AIH_ATTN_ROWS) return at_launch_rows<AtRows<DT_F16, DP>>(a, st);      \
    return kernel == AIH_ATTN_KEYS ? at_launch_keys<DT_F16, DP>(a, cus, st) : hipErrorInvalidValue; \
  }
  AIH_AT_CASE(32)
  AIH_AT_CASE(64)
  AIH_AT_CASE(96)
  AIH_AT_CASE(128)
  AIH_AT_CASE(256)
#undef AIH_AT_CASE
  return hipErrorInvalidValue;
}

}  // namespace aih
