// The fp32 instances of masked_attention_fwd.h.
#include "masked_attention_fwd.h"

namespace ffk {

template <int DP>
static hipError_t by_rows(hipStream_t st, MaskedAttnParams const &p, int groups) {
  if constexpr (DP <= 128) {  // (the tiles of four waves' keys of 256 columns are more than a CU's LDS)
    if (groups == 1) return masked_fwd_launch<float, DP, 1>(st, p);
  }
  return masked_fwd_launch<float, DP, 4>(st, p);
}

hipError_t masked_attention_fwd_f32(hipStream_t st, MaskedAttnParams const &p, int padded, int groups) {
  switch (padded) {
    case 64: return by_rows<64>(st, p, groups);
    case 96: return by_rows<96>(st, p, groups);
    case 128: return by_rows<128>(st, p, groups);
    default: return by_rows<256>(st, p, groups);
  }
}

}  // namespace ffk
