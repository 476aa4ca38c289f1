// The bf16 instances of the dK/dV kernel of masked_attention_bwd.h.
#include "masked_attention_bwd.h"

namespace ffk {

template <int DP>
static hipError_t by_parts(hipStream_t st, MaskedAttnParams const &p) {
  if constexpr (DP <= 128) {
    return masked_dkdv_launch<bf16, DP, 3>(st, p);
  } else {
    hipError_t const e = masked_dkdv_launch<bf16, DP, 1>(st, p);
    if (e != hipSuccess) return e;
    return masked_dkdv_launch<bf16, DP, 2>(st, p);
  }
}

hipError_t masked_attention_dkdv_bf16(hipStream_t st, MaskedAttnParams const &p, int padded) {
  switch (padded) {
    case 64: return by_parts<64>(st, p);
    case 96: return by_parts<96>(st, p);
    case 128: return by_parts<128>(st, p);
    default: return by_parts<256>(st, p);
  }
}

}  // namespace ffk
