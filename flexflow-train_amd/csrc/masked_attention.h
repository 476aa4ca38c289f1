// Masked attention: what its forward and backward kernels share.
//
// For batch b, query head h (which reads key head h / G, G = heads / kv_heads), query row i at position
// p_i = query_offset + i and key j:
//   x = scale q_i . k_j      s = cap tanh(x / cap)  (cap 0: x)  - slope_h |p_i - j|
//   j is seen iff lo_i <= j < hi_i   (and j <= p_i if causal)
//   P = softmax over the seen keys, O = P V, lse = log sum exp(s); a row that sees nothing: O = 0, lse = -inf
//   delta_i = O_i . dO_i     dS = P (dO V^T - delta)     dX = dS (1 - tanh^2) scale
//   dQ = dX K      dK = dX^T Q, dV = P^T dO, summed over the G heads that read the key head
// A row that sees one key has P = 1 whatever its score, so dS = 0.  dP and delta, sums of the same products in different
// orders, would leave some 2^-23 of |dO| |v| in its place, and all of dQ and dK of sequences of one position is nothing else.
// So the dQ kernels let such a row see nothing where dS is masked (score_range), and the dK/dV kernels correct P and dS of
// the tiles that have one, or, for heads, clear its Q in LDS, which with what write_row leaves of it gives P = 1.  No
// instruction for it in a loop (a comparison a score took 2 to 4 % of a capped pass over 4 x 4096 tokens).
//
// The G query heads of a key head are one longer axis of rows, r = i G + g: they share the tiles of K and V that a
// workgroup brings into LDS, the keys' gradients are sums over that one axis (no atomics), and a few query rows still
// fill an MFMA tile.  All kernels compute scores transposed or not such that a lane owns a row's (forward, dQ) or a
// key's (dK, dV) column of the 32 x 32 accumulator, and feed the accumulator to the next product from registers:
//   MFMA 32x32: A operand row l%32, B operand column l%32, both k = 8*(l/32)..+7 of a step of 16; accumulator element
//   r: row 8*(r/4) + 4*(l/32) + r%4, column l%32.  An accumulator's elements 8s..8s+7 are the k-slots of step s of
//   the next product; its other operand is read with the same permutation.  fp32 takes a step of 16 as eight
//   32x32x2 instructions on the same slots, so that both types share every index below.
#pragma once
#include "attention_common.h"

namespace ffk {

// Rows that a summary of ranges covers: the dQ kernels write one for every 32 rows, the dK/dV kernels skip by them.
struct RangeSummary {
  int lo_min, hi_max;  // every key that some row sees lies in [lo_min, hi_max)
  int lo_max, hi_min;  // every row sees all of [lo_max, hi_min); nothing is, with (1 << 30) for lo_max, where a row sees one key
};

// What the dQ kernels leave in memory of every row for the dK/dV kernels: arrays of padded_rows entries, one set for each
// (batch, key head), which a tile's rows are read from in order.  Rows behind the last one see nothing.
enum { kRowLse2 = 0, kRowDelta = 1, kRowLo = 2, kRowHi = 3, kRowSlope = 4, kRowPosition = 5, kRowFields = 6 };

struct MaskedAttnParams {
  void const *q, *k, *v;
  void *o;
  void const *d_o;
  float *lse;
  float *rows;  // [B, KH, kRowFields, padded_rows], integers by their bits
  void *dq, *dk, *dv;
  int const *ranges;    // [B, Sq, 2] or NULL
  float const *slopes;  // [H] or NULL
  RangeSummary *summary;  // [B, ceil(Sq G / 32)]
  int B, H, KH, G, Sq, Skv, Dq, Dv, R;  // R = Sq G rows of a key head
  int padded_rows;                      // R up to whole tiles of 64
  int64_t q_bs, q_ss, k_bs, k_ss, v_bs, v_ss, o_bs, o_ss;
  int q_offset;
  // A score in powers of two is  score_scale y + shift,  y = capped(raw) - slope_unit slope_h |p_i - j|  (see capped);
  // its derivative by the raw product, over ln 2, is score_scale times the derivative of capped.  What is the same for
  // all scores of a row is taken out of the loops: the shift goes into the log-sum-exp, the gradients' factor to their store.
  float score_scale, shift, slope_unit, grad_scale;
  float cap_in;
  int capped, causal;  // capped: how (see capped)
  FastDiv group, heads_div, places_div;  // by G, KH and KH B
  // forward, split over the keys: partial O (unnormalised), maximum and sum of each part
  int splits;
  float *part_o, *part_ml;
};

__device__ __forceinline__ void row_of(MaskedAttnParams const &p, int r, int &i, int &g) {
  uint32_t a, b;
  p.group.divmod((uint32_t)r, a, b);
  i = (int)a;
  g = (int)b;
}
// The key head that this workgroup works on, its batch entry and their place among all; returns the workgroup's number there.
__device__ __forceinline__ int place_of(MaskedAttnParams const &p, int &kh, int &b, int &hb) {
  uint32_t rest, place, entry, head;
  p.places_div.divmod(blockIdx.x, rest, place);
  p.heads_div.divmod(place, entry, head);
  kh = (int)head;
  b = (int)entry;
  hb = (int)place;
  return (int)rest;
}
// The keys that row i of batch b sees, within [0, Skv]; nothing is (INT_MAX / 2, 0), which widens no window.
__device__ __forceinline__ void row_range(MaskedAttnParams const &p, int b, int i, int &lo, int &hi) {
  lo = 0;
  hi = p.Skv;
  if (p.ranges != nullptr) {
    int2 const v = reinterpret_cast<int2 const *>(p.ranges)[(int64_t)b * p.Sq + i];
    lo = max(v.x, 0);
    hi = min(v.y, p.Skv);
  }
  if (p.causal) hi = min(hi, p.q_offset + i + 1);
  if (lo >= hi) {
    lo = 1 << 30;
    hi = 0;
  }
}

// Whether a range is a single key's.
__device__ __forceinline__ bool one_key(int lo, int hi) { return hi - lo == 1; }
// The keys whose scores have a gradient in a row that sees [lo, hi): all of them, or none where there is one.
__device__ __forceinline__ void score_range(int lo, int hi, int &ds_lo, int &ds_hi) {
  ds_lo = one_key(lo, hi) ? 1 << 30 : lo;
  ds_hi = one_key(lo, hi) ? 0 : hi;
}
// lo_max of a summary, of a wave whose rows see [lo, hi)
__device__ __forceinline__ int summary_lo_max(int lo, int hi, int w_lo_max) {
  return __builtin_amdgcn_ballot_w64(one_key(lo, hi)) != 0 ? 1 << 30 : w_lo_max;
}

__device__ __forceinline__ void write_row(MaskedAttnParams const &p, int b, int kh, int row, float lse2, float delta, int lo, int hi,
                                          float slope, int position) {
  if (row >= p.padded_rows) return;
  float *rows = p.rows + (int64_t)(b * p.KH + kh) * kRowFields * p.padded_rows + row;
  int64_t const n = p.padded_rows;
  bool const one = one_key(lo, hi);  // (with Q cleared y is 0, or the logistic function's 1/2: score_scale y = -shift)
  rows[kRowLse2 * n] = one ? -p.shift : lse2;
  rows[kRowDelta * n] = delta;
  rows[kRowLo * n] = __int_as_float(lo);
  rows[kRowHi * n] = __int_as_float(hi);
  if (p.slopes != nullptr) {
    rows[kRowSlope * n] = one ? 0.0f : slope;
    rows[kRowPosition * n] = __int_as_float(position);
  }
}
// the rows from `first` on that no workgroup of the dQ kernel owns
__device__ __forceinline__ void write_padding(MaskedAttnParams const &p, int b, int kh, int first, int t) {
  for (int row = first + t; row < p.padded_rows; row += 256) write_row(p, b, kh, row, 0.0f, 0.0f, 1 << 30, 0, 0.0f, 0);
}

// bf16: the longest window of keys in which a workgroup of the dQ kernels takes delta from P and dP themselves, in a pass over
// the keys of its own, in place of from O as it was stored.  O's rounding reaches dS times what a single key holds of O: rows of few
// keys lose most (dQ and dK of 5 causal tokens with scores to 12: 0.006 of their size off, 0.0027 from P and dP; of
// 300 tokens 0.0038).  The pass costs two products more: up to 128 keys nothing that a call shows, up to 256 a fifth of
// dQ for documents of that length (8 x 512 tokens, 16 heads of 64: 21 and 25 us).
constexpr int kExactDelta = 128;

// ---- one step of 16 of a product, for either type -------------------------
template <typename T>
struct Frag;
template <>
struct Frag<bf16> {
  bf16x8 v;
};
template <>
struct Frag<float> {
  f32x4 a, b;
};
__device__ __forceinline__ void mma(f32x16 &acc, Frag<bf16> const &a, Frag<bf16> const &b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16 &acc, Frag<float> const &a, Frag<float> const &b) {
#pragma unroll
  for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.a[j], b.a[j], acc, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.b[j], b.b[j], acc, 0, 0, 0);
}
// 8 elements from d0 on of a row in memory, zeros past the head size D (a multiple of 8, fp32: of 4)
__device__ __forceinline__ Frag<bf16> frag_row(bf16 const *row, int d0, int D) {
  union {
    u32x4 u;
    bf16x8 b;
  } x;
  x.u = u32x4{0u, 0u, 0u, 0u};
  if (d0 < D) x.u = *reinterpret_cast<u32x4 const *>(row + d0);
  return Frag<bf16>{x.b};
}
__device__ __forceinline__ Frag<float> frag_row(float const *row, int d0, int D) {
  Frag<float> f = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
  if (d0 < D) f.a = *reinterpret_cast<f32x4 const *>(row + d0);
  if (d0 + 4 < D) f.b = *reinterpret_cast<f32x4 const *>(row + d0 + 4);
  return f;
}
// 8 elements of a row of an LDS tile
__device__ __forceinline__ Frag<bf16> frag_lds(bf16 const *p) { return Frag<bf16>{*reinterpret_cast<bf16x8 const *>(p)}; }
__device__ __forceinline__ Frag<float> frag_lds(float const *p) {
  return Frag<float>{*reinterpret_cast<f32x4 const *>(p), *reinterpret_cast<f32x4 const *>(p + 4)};
}
// The slots of step s of an accumulator whose rows are the tile's rows, down the columns col0 + l%32: `tile` points at
// the lane's place (turn_off) of the tile's first row.
template <typename T>
__device__ __forceinline__ int turn_off(int stride, int lane);
template <>
__device__ __forceinline__ int turn_off<bf16>(int stride, int lane) { return lane_tr_off(stride, lane); }
template <>
__device__ __forceinline__ int turn_off<float>(int stride, int lane) { return 4 * (lane >> 5) * stride + (lane & 31); }
__device__ __forceinline__ Frag<bf16> frag_turned(bf16 const *tile, int stride, int s, int col0) {
  return Frag<bf16>{frag_tr_acc(tile, stride, 0, s, col0)};
}
__device__ __forceinline__ Frag<float> frag_turned(float const *tile, int stride, int s, int col0) {
  Frag<float> f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    f.a[j] = tile[(16 * s + j) * stride + col0];
    f.b[j] = tile[(16 * s + 8 + j) * stride + col0];
  }
  return f;
}
__device__ __forceinline__ Frag<bf16> frag_acc(float const *v, bf16 const *) { return Frag<bf16>{pack8(v)}; }
__device__ __forceinline__ Frag<float> frag_acc(float const *v, float const *) {
  return Frag<float>{{v[0], v[1], v[2], v[3]}, {v[4], v[5], v[6], v[7]}};
}

// Row strides of LDS tiles, in elements.  A tile that is read by rows (16 bytes a lane, 16 rows at a time) wants rows
// 4 banks apart, one that is read turned (bf16: 4 rows x 64 bytes) 16 banks apart, one that is read both ways 20.
template <typename T, int DP>
struct TileStride {
  static constexpr int row = sizeof(T) == 2 ? DP + 8 : DP + 4;
  static constexpr int turned = sizeof(T) == 2 ? (DP % 64 == 0 ? DP + 32 : DP) : DP + 4;
  static constexpr int both = sizeof(T) == 2 ? (DP % 64 == 0 ? DP + 40 : DP + 8) : DP + 4;
};

// A tile of N rows on its way from memory to LDS.  Columns past the head size become zeros on the way into LDS (a lane
// there fetches the row's first columns again: no branch around a load), rows outside of the tensors are the caller's to
// replace by others: whatever lies in memory that no row of the workgroup sees is not read.
template <typename T, int DP, int N>
struct TileRegs {
  static constexpr int kE = 16 / (int)sizeof(T);  // elements of a 16-byte chunk
  static constexpr int kCPR = DP / kE;
  static constexpr int kN = (N * kCPR + 255) / 256;
  u32x4 r[kN];
  template <typename ROW>
  __device__ __forceinline__ void load(ROW row_pointer, int D, int t) {
#pragma unroll
    for (int n = 0; n < kN; n++) {
      int const c = t + n * 256, row = c / kCPR, ch = c % kCPR;
      r[n] = *reinterpret_cast<u32x4 const *>(row_pointer(row) + (ch * kE < D ? ch * kE : 0));
    }
  }
  // `keep(n)`: whether the row of chunk n is wanted, or zeros in its place
  template <typename KEEP>
  __device__ __forceinline__ void store(T *tile, int stride, int D, int t, KEEP keep) const {
#pragma unroll
    for (int n = 0; n < kN; n++) {
      int const c = t + n * 256, row = c / kCPR, ch = c % kCPR;
      u32x4 const v = ch * kE < D && keep(n) ? r[n] : u32x4{0u, 0u, 0u, 0u};
      if (N * kCPR % 256 == 0 || c < N * kCPR) *reinterpret_cast<u32x4 *>(tile + row * stride + ch * kE) = v;
    }
  }
  __device__ __forceinline__ void store(T *tile, int stride, int D, int t) const {
    store(tile, stride, D, t, [](int) { return true; });
  }
};

// The cap's part of a score that is not linear, and its derivative (1 without a cap, where y is the raw product), two ways.
//   kCapTanh: y = tanh(scale raw / cap), score_scale = cap log2(e), derivative 1 - y^2, by the library's tanh, a few 2^-24 of
//   itself off.
//   kCapLogistic: y = 1 / (1 + 2^(cap_in raw)), cap_in = -2 log2(e) scale / cap, on the hardware's exponential and reciprocal:
//   tanh is 2 y - 1, so score_scale = 2 cap log2(e), shift = -cap log2(e), and 1 - tanh^2 = 4 (y - y^2), of which grad_scale has
//   the 4.  Four vector instructions a score and two for the derivative.  Scores next to nothing are next to y = 1/2, where a
//   step of y is 2^-24, so this one is off by up to 2^-21 cap whatever the score.
// bf16 takes the second up to a cap of kLogisticCap, 6e-5 there and 2e-5 at 50, far below what bf16 scores carry;
// past it (at 10^5 scores would be 0.01 off, at 10^8 all the same) the first one, in the general kernels: 4 x 2048 tokens,
// 16 heads of 128 on 4, causal, 1003 us with gradients, and 506 at a cap of 100.  fp32 takes the first: its products take
// sixteen times as long.
enum { kNoCap = 0, kCapLogistic = 1, kCapTanh = 2 };
constexpr float kLogisticCap = 128.0f;
template <int CAP>
__device__ __forceinline__ float capped(MaskedAttnParams const &p, float raw) {
  if constexpr (CAP == kNoCap) return raw;
  else if constexpr (CAP == kCapLogistic) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(raw * p.cap_in));
  else return tanhf(raw * p.cap_in);
}
template <int CAP>
__device__ __forceinline__ float capped_slope(float y) {
  return CAP == kCapLogistic ? __builtin_fmaf(-y, y, y) : __builtin_fmaf(-y, y, 1.0f);
}

// The general kernels' instances: launch(how the score is capped, and 4 with a bias).
template <typename T, typename LAUNCH>
static hipError_t masked_by_score(MaskedAttnParams const &p, LAUNCH launch) {
  auto const either = [&](auto cap) {
    constexpr int kCap = decltype(cap)::value;
    return p.slopes != nullptr ? launch(std::integral_constant<int, kCap | 4>{}) : launch(std::integral_constant<int, kCap>{});
  };
  if constexpr (sizeof(T) == 2) {
    if (p.capped == kCapLogistic) return either(std::integral_constant<int, kCapLogistic>{});
  }
  return p.capped != kNoCap ? either(std::integral_constant<int, kCapTanh>{}) : either(std::integral_constant<int, kNoCap>{});
}

// A wave's smallest and largest of an integer, scalar.
__device__ __forceinline__ int wave_min_int(int v) {
  return __builtin_amdgcn_readfirstlane(wave_reduce(v, [](int a, int b) { return min(a, b); }));
}
__device__ __forceinline__ int wave_max_int(int v) {
  return __builtin_amdgcn_readfirstlane(wave_reduce(v, [](int a, int b) { return max(a, b); }));
}

// acc += a b on an accumulator that stays in accumulation registers: left to itself the compiler keeps some of a wave's
// values in the wrong kind of register and moves them there and back in every tile.  It does not see that results take
// time: mma_settled has to stand between the last of these and any other use of an accumulator, and four wait states
// between a vector instruction that writes an operand or an accumulator and the next of these
// (tests/test_masked_accumulators.py reads the built library for both).
__device__ __forceinline__ void mma_kept(f32x16 &acc, bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
template <int N>
__device__ __forceinline__ void mma_settled(f32x16 (&acc)[N]) {
  asm volatile("s_nop 15\n\ts_nop 7" ::);
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+a"(acc[i]));
}

// Writes 4 consecutive elements.
__device__ __forceinline__ void store4(bf16 *p, float a, float b, float c, float d) {
  *reinterpret_cast<u32x2 *>(p) = u32x2{pack_bf16x2(a, b), pack_bf16x2(c, d)};
}
__device__ __forceinline__ void store4(float *p, float a, float b, float c, float d) {
  *reinterpret_cast<f32x4 *>(p) = f32x4{a, b, c, d};
}

}  // namespace ffk
