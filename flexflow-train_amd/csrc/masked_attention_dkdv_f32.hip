// The fp32 instances of the dK/dV kernel of masked_attention_bwd.h.
#include "masked_attention_bwd.h"

namespace ffk {

template <int DP>
static hipError_t by_parts(hipStream_t st, MaskedAttnParams const &p, bool extra) {
  if constexpr (DP <= 128) {
    return extra ? masked_dkdv_launch<float, DP, 3, true>(st, p) : masked_dkdv_launch<float, DP, 3, false>(st, p);
  } else {
    hipError_t const e = extra ? masked_dkdv_launch<float, DP, 1, true>(st, p) : masked_dkdv_launch<float, DP, 1, false>(st, p);
    if (e != hipSuccess) return e;
    return extra ? masked_dkdv_launch<float, DP, 2, true>(st, p) : masked_dkdv_launch<float, DP, 2, false>(st, p);
  }
}

hipError_t masked_attention_dkdv_f32(hipStream_t st, MaskedAttnParams const &p, int padded, bool extra) {
  switch (padded) {
    case 64: return by_parts<64>(st, p, extra);
    case 96: return by_parts<96>(st, p, extra);
    case 128: return by_parts<128>(st, p, extra);
    default: return by_parts<256>(st, p, extra);
  }
}

}  // namespace ffk
