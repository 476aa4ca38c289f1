// The bf16 instances of masked_attention_fwd.h.
#include "masked_attention_fwd.h"

namespace ffk {

template <int DP>
static hipError_t by_rows(hipStream_t st, MaskedAttnParams const &p, int groups) {
  if (groups == 1) return masked_fwd_launch<bf16, DP, 1>(st, p);
  return masked_fwd_launch<bf16, DP, 4>(st, p);
}

hipError_t masked_attention_fwd_bf16(hipStream_t st, MaskedAttnParams const &p, int padded, int groups) {
  switch (padded) {
    case 64: return by_rows<64>(st, p, groups);
    case 96: return by_rows<96>(st, p, groups);
    case 128: return by_rows<128>(st, p, groups);
    default: return by_rows<256>(st, p, groups);
  }
}

}  // namespace ffk
