// What the kernels for bf16 heads up to 128 share: heads that lie in LDS at a pitch of 64 or 128 elements.
//
// Heads of other sizes (PAD) are made longer with zeros on the way: a 16-byte chunk behind the head's end is asked for
// beyond the descriptor's last byte, which costs no memory access and leaves zeros in LDS, so nothing of the next head or
// row enters a product; those columns are not stored.  U is how many elements of the pitch are computed with: 96 of 128
// where heads end there.
#pragma once
#include "masked_attention.h"
#include "lds_dma.h"

namespace ffk {

constexpr unsigned kBehind = 0x80000000u;  // PAD: the descriptors' length, and the offset of what is to be zero

template <bool PAD>
__device__ __forceinline__ i32x4 tile_resource(bf16 const *p) {
  return buffer_resource(p, PAD ? kBehind : 0xffffffffu);
}
// The byte offset of element `column` (a multiple of 8) of a row whose first element is `first`.
template <bool PAD>
__device__ __forceinline__ unsigned tile_offset(int64_t first, int column, int dim) {
  unsigned const at = (unsigned)(first + column) * 2u;
  return PAD && column >= dim ? kBehind : at;
}
// The same for head g of a row at `row_bytes`.
template <bool PAD>
__device__ __forceinline__ unsigned row_offset(unsigned row_bytes, int g, int column, int dim) {
  unsigned const at = row_bytes + (unsigned)(g * dim + column) * 2u;
  return PAD && column >= dim ? kBehind : at;
}
// Eight elements of a head in memory, or zeros behind it.
template <bool PAD>
__device__ __forceinline__ bf16x8 head_chunk(bf16 const *head, int column, int dim) {
  if constexpr (PAD) {
    if (column >= dim) return bf16x8{};
  }
  return *reinterpret_cast<bf16x8 const *>(head + column);
}

}  // namespace ffk
