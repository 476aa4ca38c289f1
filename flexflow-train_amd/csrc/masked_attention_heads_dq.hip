// Masked attention, dQ for bf16 heads of 64 and 128 (see masked_attention.h for the mathematics and layouts).
//
// One workgroup owns 128 rows of one key head, 32 to a wave, whose Q and dO rows are MFMA operands in registers; two
// workgroups run on a CU, so that the vector work of one covers the matrix work of the other.  Keys and values come in
// tiles of 32, through registers into two LDS buffers, two tiles ahead.  Like the general kernel it leaves delta, the
// log-sum-exp and the ranges of its rows in memory for the dK/dV kernel, and summaries of the ranges.
#include "masked_attention.h"

namespace ffk {

template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) void masked_dq_heads_kernel(MaskedAttnParams p) {
  constexpr int kT = 32, kStride = D + 40;  // serves 16-byte and transposing reads
  constexpr int kChunks = kT * D / 8 / 256;
  __shared__ __attribute__((aligned(16))) bf16 Ks[2][kT * kStride];
  __shared__ __attribute__((aligned(16))) bf16 Vs[2][kT * kStride];
  __shared__ int window[2][4];
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const nrb = (p.R + 127) / 128;
  int const hb = blockIdx.x % (p.KH * p.B);
  int const rb = nrb - 1 - blockIdx.x / (p.KH * p.B);
  int const kh = hb % p.KH, b = hb / p.KH;
  int const row0 = rb * 128 + wave * 32;
  int const row = row0 + (lane & 31);
  int qi, qg;
  row_of(p, min(row, p.R - 1), qi, qg);
  int const head = kh * p.G + qg;
  int lo, hi;
  row_range(p, b, qi, lo, hi);
  if (row >= p.R) {
    lo = 1 << 30;
    hi = 0;
  }
  int64_t const q_at = (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * D;
  int64_t const o_at = (int64_t)b * p.o_bs + (int64_t)qi * p.o_ss + (int64_t)head * D;
  bf16 const *qp = static_cast<bf16 const *>(p.q) + q_at, *gp = static_cast<bf16 const *>(p.d_o) + o_at;
  bf16 const *op = static_cast<bf16 const *>(p.o) + o_at;
  bf16 const *kp = static_cast<bf16 const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * D;
  bf16 const *vp = static_cast<bf16 const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * D;
  bf16x8 qf[D / 16], gf[D / 16];
  float part = 0.0f;
#pragma unroll
  for (int kk = 0; kk < D / 16; kk++) {
    qf[kk] = *reinterpret_cast<bf16x8 const *>(qp + kk * 16 + h32 * 8);
    gf[kk] = *reinterpret_cast<bf16x8 const *>(gp + kk * 16 + h32 * 8);
    bf16x8 const of = *reinterpret_cast<bf16x8 const *>(op + kk * 16 + h32 * 8);
#pragma unroll
    for (int e = 0; e < 8; e++) part += (float)of[e] * (float)gf[kk][e];
  }
  float const delta = part + __shfl_xor(part, 32, 64);
  float const lse2 = p.lse[((int64_t)b * p.H + head) * p.Sq + qi] * kLog2e - p.shift;
  float slope = 0.0f;
  if constexpr (BIAS) slope = p.slopes[head] * p.slope_unit;
  int const position = p.q_offset + qi;

  int const w_lo_min = wave_min_int(lo), w_hi_max = wave_max_int(hi), w_lo_max = wave_max_int(lo), w_hi_min = wave_min_int(hi);
  if (h32 == 0) write_row(p, b, kh, row, lse2, delta, lo, hi, slope, position);
  if (lane == 0) {
    window[0][wave] = w_lo_min;
    window[1][wave] = w_hi_max;
    if (kh == 0 && row0 < p.R)
      p.summary[(int64_t)b * ((p.R + 31) / 32) + row0 / 32] = RangeSummary{w_lo_min, w_hi_max, w_lo_max, w_hi_min};
  }
  __syncthreads();
  int const lo_all = __builtin_amdgcn_readfirstlane(min(min(window[0][0], window[0][1]), min(window[0][2], window[0][3])));
  int const hi_all = __builtin_amdgcn_readfirstlane(max(max(window[1][0], window[1][1]), max(window[1][2], window[1][3])));
  int const ntiles = hi_all > lo_all ? (hi_all - lo_all + kT - 1) / kT : 0;

  f32x16 dq[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) dq[i][r] = 0.0f;

  if (ntiles > 0) {
    u32x4 rk[2][kChunks], rv[2][kChunks];
    auto gload = [&](int kt0, auto set_tag) {
      constexpr int R = decltype(set_tag)::value;
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        int const c = t + i * 256;
        int const r = c / (D / 8), ch = c % (D / 8);
        int const gr = min(kt0 + r, hi_all - 1);  // what no row of the workgroup sees is not read
        rk[R][i] = *reinterpret_cast<u32x4 const *>(kp + (int64_t)gr * p.k_ss + ch * 8);
        rv[R][i] = *reinterpret_cast<u32x4 const *>(vp + (int64_t)gr * p.v_ss + ch * 8);
      }
    };
    auto lstore = [&](auto set_tag) {
      constexpr int R = decltype(set_tag)::value;
#pragma unroll
      for (int i = 0; i < kChunks; i++) {
        int const c = t + i * 256;
        int const r = c / (D / 8), ch = c % (D / 8);
        *reinterpret_cast<u32x4 *>(&Ks[R][r * kStride + ch * 8]) = rk[R][i];
        *reinterpret_cast<u32x4 *>(&Vs[R][r * kStride + ch * 8]) = rv[R][i];
      }
    };
    using Set0 = std::integral_constant<int, 0>;
    using Set1 = std::integral_constant<int, 1>;
    int const koff = lane_k_off(kStride, lane);
    int const toff = lane_tr_off(kStride, lane);
    gload(lo_all, Set0{});
    lstore(Set0{});
    gload(lo_all + kT, Set1{});  // unconditional, like every load ahead below: the loop's waits are exact then
    __syncthreads();
    auto step = [&](int it, auto parity) {
      constexpr int cur = decltype(parity)::value;  // == it % 2
      int const kt0 = lo_all + it * kT;
      gload(kt0 + 2 * kT, parity);
      if (it < ntiles && kt0 < w_hi_max && kt0 + kT > w_lo_min) {
        bf16 const *kk_ = Ks[cur] + koff, *vk_ = Vs[cur] + koff, *ktr = Ks[cur] + toff;
        // S^T = K Q^T, dP^T = V dO^T: rows = keys of the tile, column = row
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[r] = 0.0f;
          dp[r] = 0.0f;
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_k(kk_, kStride, 0, kk * 16), qf[kk], s, 0, 0, 0);
          dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_k(vk_, kStride, 0, kk * 16), gf[kk], dp, 0, 0, 0);
        }
        float const distance = (float)(position - (kt0 + 4 * h32));
        float ds[16];
#pragma unroll
        for (int r = 0; r < 16; r++) {
          float const y = capped<bf16, CAP>(p, s[r]);
          float x = y;
          if constexpr (BIAS) x = __builtin_fmaf(-slope, fabsf(distance - (float)(8 * (r >> 2) + (r & 3))), x);
          ds[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, p.score_scale, -lse2)) * (dp[r] - delta);
          if constexpr (CAP) ds[r] *= capped_slope<bf16>(y);
        }
        if (kt0 < w_lo_max || kt0 + kT > w_hi_min) {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            int const kv = kt0 + 8 * (r >> 2) + 4 * h32 + (r & 3);
            ds[r] = kv < lo || kv >= hi ? 0.0f : ds[r];
          }
        }
        // dQ^T += K^T dS^T : A = K^T (rows d) by transposing loads, B = dS^T
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
          bf16x8 const db = pack8(ds + 8 * s2);
#pragma unroll
          for (int i = 0; i < D / 32; i++)
            dq[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_acc(ktr, kStride, 0, s2, i * 32), db, dq[i], 0, 0, 0);
        }
      }
      if (it + 1 < ntiles) lstore(std::integral_constant<int, cur ^ 1>{});
      __syncthreads();
    };
    // in pairs (an odd count runs one idle step)
    for (int it = 0; it < ntiles; it += 2) {
      step(it, Set0{});
      step(it + 1, Set1{});
    }
  }

  if (row < p.R) {
    bf16 *dqp = static_cast<bf16 *>(p.dq) + q_at;
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        store4(dqp + i * 32 + 8 * g + 4 * h32, dq[i][4 * g] * p.grad_scale, dq[i][4 * g + 1] * p.grad_scale, dq[i][4 * g + 2] * p.grad_scale,
               dq[i][4 * g + 3] * p.grad_scale);
  }
}

template <int D>
static void launch(hipStream_t st, MaskedAttnParams const &p) {
  dim3 const grid((unsigned)(ceil_div(p.R, 128) * p.KH * p.B));
  bool const cap = p.capped != 0, bias = p.slopes != nullptr;
  if (cap && bias) masked_dq_heads_kernel<D, true, true><<<grid, 256, 0, st>>>(p);
  else if (cap) masked_dq_heads_kernel<D, true, false><<<grid, 256, 0, st>>>(p);
  else if (bias) masked_dq_heads_kernel<D, false, true><<<grid, 256, 0, st>>>(p);
  else masked_dq_heads_kernel<D, false, false><<<grid, 256, 0, st>>>(p);
}

hipError_t masked_attention_dq_heads(hipStream_t st, MaskedAttnParams const &p) {
  if (p.Dq == 64) launch<64>(st, p);
  else launch<128>(st, p);
  return hipGetLastError();
}

}  // namespace ffk
