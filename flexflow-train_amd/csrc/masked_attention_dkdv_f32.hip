// The fp32 instances of the dK/dV kernel of masked_attention_bwd.h.
#include "masked_attention_bwd.h"

namespace ffk {

template <int DP, int KG>
static hipError_t by_parts(hipStream_t st, MaskedAttnParams const &p) {
  if constexpr (DP <= 128) {
    return masked_dkdv_launch<float, DP, KG, 3>(st, p);
  } else {
    hipError_t const e = masked_dkdv_launch<float, DP, KG, 1>(st, p);
    return e != hipSuccess ? e : masked_dkdv_launch<float, DP, KG, 2>(st, p);
  }
}
template <int DP>
static hipError_t by_keys(hipStream_t st, MaskedAttnParams const &p, int groups) {
  if constexpr (DP <= 128) {  // (past that the tiles of four waves' rows leave no registers, or no LDS)
    if (groups == 1) return by_parts<DP, 1>(st, p);
  }
  return by_parts<DP, 4>(st, p);
}

hipError_t masked_attention_dkdv_f32(hipStream_t st, MaskedAttnParams const &p, int padded, int groups) {
  switch (padded) {
    case 64: return by_keys<64>(st, p, groups);
    case 96: return by_keys<96>(st, p, groups);
    case 128: return by_keys<128>(st, p, groups);
    default: return by_keys<256>(st, p, groups);
  }
}

}  // namespace ffk
