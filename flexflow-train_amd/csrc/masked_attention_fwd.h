// Masked attention, forward: any head size, either type (see masked_attention.h for the mathematics and layouts).
// A template that masked_attention_fwd_*.hip instantiate, so that they compile side by side.
//
// One workgroup takes 32 RG rows of one (batch, key head): RG groups of 32 rows, whose KW = 4 / RG waves take the keys in
// turn (their sums meet in LDS at the end).  Keys and values pass through LDS in tiles of 32 J KW rows, the next tile
// on its way in registers meanwhile.  The loop runs over the union of the rows' ranges only; a wave skips a tile that none
// of its rows sees, and compares ranges element by element only where a tile is not seen whole by all of them.
//   bf16 heads of 256, 4 x 2000 tokens, 8 heads on 4, causal: 158 us (0.41 PFLOP/s), bound by LDS reads and one wave to a SIMD;
// fp32, 4 x 2000 tokens, 8 heads of 64, causal: 214 us (77 TFLOP/s), half the rate of the fp32 matrix instructions, of which
// masked tiles at the diagonal take some, and single-element reads of V's turned fragments the rest or not: not measured.
#pragma once
#include "masked_attention.h"

namespace ffk {

template <typename T, int DP, int RG>
struct MaskedFwd {
  static constexpr int kKW = 4 / RG;
  static constexpr int kJ = sizeof(T) == 2 && RG == 4 && DP <= 128 ? 2 : 1;  // 32-key blocks of a wave and tile
  static constexpr int kT = 32 * kJ * kKW;
  static constexpr int kKS = TileStride<T, DP>::row, kVS = TileStride<T, DP>::turned;
  static constexpr int kTile = kT * (kKS + kVS) * (int)sizeof(T);
  static constexpr int kBuffers = 2 * kTile <= 152 * 1024 ? 2 : 1;
  static constexpr int kMerge = (kKW - 1) * RG * (DP * 32 + 128) * 4;
  static constexpr int kBytes = kBuffers * kTile > kMerge ? kBuffers * kTile : kMerge;
  static_assert(kBytes <= 156 * 1024, "LDS of a CU");
};

template <typename T, int DP, int RG, int EXTRA>
__global__ __launch_bounds__(256) void masked_fwd_kernel(MaskedAttnParams p) {
  using C = MaskedFwd<T, DP, RG>;
  constexpr int J = C::kJ, KW = C::kKW;
  constexpr int kCap = EXTRA & 3;  // kNoCap, kCapLogistic or kCapTanh
  constexpr bool kBias = (EXTRA & 4) != 0;
  extern __shared__ __attribute__((aligned(16))) uint8_t pool[];
  __shared__ int window[2][4];
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const qw = wave / KW, kw = wave % KW;
  int const nrb = (p.R + 32 * RG - 1) / (32 * RG);
  int kh, b, hb;
  int const rest = place_of(p, kh, b, hb);
  int const split = rest % p.splits;
  int const rb = nrb - 1 - rest / p.splits;  // under a causal mask the heaviest rows go first
  int const row0 = rb * 32 * RG + qw * 32;
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
  int const w_lo_min = wave_min_int(lo), w_hi_max = wave_max_int(hi);
  // rows that see nothing make these useless bounds, which only costs comparisons
  int const w_lo_max = wave_max_int(row < p.R ? lo : 0), w_hi_min = wave_min_int(row < p.R ? hi : 1 << 30);
  if (lane == 0) {
    window[0][wave] = w_lo_min;
    window[1][wave] = w_hi_max;
  }
  __syncthreads();
  int const lo_all = __builtin_amdgcn_readfirstlane(min(min(window[0][0], window[0][1]), min(window[0][2], window[0][3])));
  int const hi_all = __builtin_amdgcn_readfirstlane(max(max(window[1][0], window[1][1]), max(window[1][2], window[1][3])));
  // this part of the window, in whole tiles
  int const all_tiles = hi_all > lo_all ? (hi_all - lo_all + C::kT - 1) / C::kT : 0;
  int const per = (all_tiles + p.splits - 1) / p.splits;
  int const first_tile = min(split * per, all_tiles), ntiles = min(per, all_tiles - first_tile);
  int const begin = lo_all + first_tile * C::kT;

  T const *qp = static_cast<T const *>(p.q) + (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * p.Dq;
  T const *kp = static_cast<T const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * p.Dq;
  T const *vp = static_cast<T const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * p.Dv;
  float const slope = kBias ? p.slopes[head] * p.slope_unit : 0.0f;
  int const position = p.q_offset + qi;

  Frag<T> qf[DP / 16];
#pragma unroll
  for (int kk = 0; kk < DP / 16; kk++) qf[kk] = frag_row(qp, kk * 16 + h32 * 8, p.Dq);
  f32x16 oacc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) oacc[i][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;

  auto k_tile = [&](int buf) { return reinterpret_cast<T *>(pool + buf * C::kTile); };
  auto v_tile = [&](int buf) { return k_tile(buf) + C::kT * C::kKS; };
  TileRegs<T, DP, C::kT> tk, tv;
  auto fetch = [&](int kv0) {
    tk.load([&](int r) { return kp + (int64_t)min(kv0 + r, hi_all - 1) * p.k_ss; }, p.Dq, t);
    tv.load([&](int r) { return vp + (int64_t)min(kv0 + r, hi_all - 1) * p.v_ss; }, p.Dv, t);
  };
  auto stash = [&](int buf) {
    tk.store(k_tile(buf), C::kKS, p.Dq, t);
    tv.store(v_tile(buf), C::kVS, p.Dv, t);
  };
  int const koff = lane_k_off(C::kKS, lane), toff = turn_off<T>(C::kVS, lane);
  if (ntiles > 0) {
    fetch(begin);
    stash(0);
  }
  __syncthreads();
  int cur = 0;
  for (int it = 0; it < ntiles; it++) {
    bool const more = it + 1 < ntiles;
    if (more) fetch(begin + (it + 1) * C::kT);
    int const kv0 = begin + it * C::kT + kw * 32 * J;  // this wave's keys
    if (kv0 < w_hi_max && kv0 + 32 * J > w_lo_min) {
      T const *kt = k_tile(cur) + kw * 32 * J * C::kKS + koff;
      T const *vt = v_tile(cur) + kw * 32 * J * C::kVS + toff;
      f32x16 s[J];
#pragma unroll
      for (int j = 0; j < J; j++) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[j][r] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) mma(s[j], frag_lds(kt + j * 32 * C::kKS + kk * 16), qf[kk]);
      }
      float const distance = (float)(position - (kv0 + 4 * h32));
#pragma unroll
      for (int j = 0; j < J; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[j][r] = capped<kCap>(p, s[j][r]);
          if constexpr (kBias) s[j][r] = __builtin_fmaf(-slope, fabsf(distance - (float)(j * 32 + 8 * (r >> 2) + (r & 3))), s[j][r]);
        }
      if (kv0 < w_lo_max || kv0 + 32 * J > w_hi_min) {
#pragma unroll
        for (int j = 0; j < J; j++) {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            int const kv = kv0 + j * 32 + 8 * (r >> 2) + 4 * h32 + (r & 3);
            if (kv < lo || kv >= hi) s[j][r] = -INFINITY;
          }
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < J; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[j][r]);
      // (score_scale is positive, so it commutes with the maximum)
      float const m_new = fmaxf(m_run, max_across_halves(mx) * p.score_scale);
      float const m_use = m_new == -INFINITY ? 0.0f : m_new;  // nothing seen yet: every exponential is 0
      float const alpha = __builtin_amdgcn_exp2f(m_run - m_use);
      float sum = 0.0f;
      Frag<T> pf[2 * J];
#pragma unroll
      for (int j = 0; j < J; j++) {
        float pv[16];
#pragma unroll
        for (int r = 0; r < 16; r++) {
          pv[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], p.score_scale, -m_use));
          sum += pv[r];
        }
        pf[2 * j] = frag_acc(pv, vp);
        pf[2 * j + 1] = frag_acc(pv + 8, vp);
      }
      l_run = l_run * alpha + sum;
      m_run = m_new;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
        for (int i = 0; i < DP / 32; i++)
#pragma unroll
          for (int r = 0; r < 16; r++) oacc[i][r] *= alpha;
      }
#pragma unroll
      for (int js = 0; js < 2 * J; js++)
#pragma unroll
        for (int i = 0; i < DP / 32; i++) mma(oacc[i], frag_turned(vt, C::kVS, js, i * 32), pf[js]);
    }
    if constexpr (C::kBuffers == 2) {
      if (more) stash(cur ^ 1);
      __syncthreads();
      cur ^= 1;
    } else {
      __syncthreads();  // every wave is done with the tile
      if (more) stash(0);
      __syncthreads();
    }
  }

  l_run += __shfl_xor(l_run, 32, 64);
  if constexpr (KW > 1) {
    // the waves of a group: O and (m, l) of the others to LDS, the first one adds them up
    float *const area = reinterpret_cast<float *>(pool);
    constexpr int kArea = DP * 32 + 128;
    __syncthreads();
    if (kw > 0) {
      float *to = area + ((kw - 1) * RG + qw) * kArea;
#pragma unroll
      for (int i = 0; i < DP / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) to[(i * 16 + r) * 64 + lane] = oacc[i][r];
      if (h32 == 0) {
        to[DP * 32 + lane] = m_run;
        to[DP * 32 + 32 + lane] = l_run;
      }
    }
    __syncthreads();
    if (kw > 0) return;
    float m_all = m_run;
#pragma unroll
    for (int w = 0; w < KW - 1; w++) m_all = fmaxf(m_all, area[(w * RG + qw) * kArea + DP * 32 + (lane & 31)]);
    float const m_use = m_all == -INFINITY ? 0.0f : m_all;
    float const f0 = __builtin_amdgcn_exp2f(m_run - m_use);
    l_run *= f0;
#pragma unroll
    for (int i = 0; i < DP / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) oacc[i][r] *= f0;
#pragma unroll
    for (int w = 0; w < KW - 1; w++) {
      float const *from = area + (w * RG + qw) * kArea;
      float const f = __builtin_amdgcn_exp2f(from[DP * 32 + (lane & 31)] - m_use);
      l_run += from[DP * 32 + 32 + (lane & 31)] * f;
#pragma unroll
      for (int i = 0; i < DP / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[i][r] += from[(i * 16 + r) * 64 + lane] * f;
    }
    m_run = m_all;
  }
  if (row >= p.R) return;
  if (p.splits > 1) {
    int64_t const at = ((int64_t)split * p.B * p.KH + hb) * p.R + row;
    float *po = p.part_o + at * p.Dv;
#pragma unroll
    for (int i = 0; i < DP / 32; i++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        int const d = i * 32 + 8 * g + 4 * h32;
        if (d < p.Dv) store4(po + d, oacc[i][4 * g], oacc[i][4 * g + 1], oacc[i][4 * g + 2], oacc[i][4 * g + 3]);
      }
    if (h32 == 0) {
      p.part_ml[2 * at] = m_run;
      p.part_ml[2 * at + 1] = l_run;
    }
    return;
  }
  float const inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
  T *op = static_cast<T *>(p.o) + (int64_t)b * p.o_bs + (int64_t)qi * p.o_ss + (int64_t)head * p.Dv;
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      int const d = i * 32 + 8 * g + 4 * h32;
      if (d < p.Dv)
        store4(op + d, oacc[i][4 * g] * inv, oacc[i][4 * g + 1] * inv, oacc[i][4 * g + 2] * inv, oacc[i][4 * g + 3] * inv);
    }
  if (h32 == 0 && p.lse != nullptr)
    p.lse[((int64_t)b * p.H + head) * p.Sq + qi] = l_run == 0.0f ? -INFINITY : (m_run + p.shift + __log2f(l_run)) * kLn2;
}

template <typename T, int DP, int RG, int EXTRA>
static hipError_t masked_fwd_launch_as(hipStream_t st, MaskedAttnParams const &p) {
  static LdsOptIn opt_in;
  using C = MaskedFwd<T, DP, RG>;
  auto kernel = &masked_fwd_kernel<T, DP, RG, EXTRA>;
  hipError_t e = opt_in.ensure(reinterpret_cast<void const *>(kernel), C::kBytes);
  if (e != hipSuccess) return e;
  int64_t const grid = ceil_div(p.R, 32 * RG) * p.splits * p.KH * p.B;
  kernel<<<dim3((unsigned)grid), 256, C::kBytes, st>>>(p);
  return hipGetLastError();
}

template <typename T, int DP, int RG>
static hipError_t masked_fwd_launch(hipStream_t st, MaskedAttnParams const &p) {
  return masked_by_score<T>(p, [&](auto extra) { return masked_fwd_launch_as<T, DP, RG, decltype(extra)::value>(st, p); });
}

}  // namespace ffk
