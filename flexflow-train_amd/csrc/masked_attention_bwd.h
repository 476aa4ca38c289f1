// Masked attention, backward: any head size, either type (see masked_attention.h for the mathematics and layouts).
// Templates that masked_attention_{dq,dkdv}_*.hip instantiate, so that they compile side by side.
//
// Two kernels without atomics, both of which compute P again from the saved log-sum-exp.  The dQ kernel owns 32 RG rows
// and runs over the keys in their ranges; it also leaves delta = rowsum(O dO) = rowsum(P dP) and, for every 32 rows, a summary of their
// ranges in memory for the dK/dV kernel, which runs behind it.  That one owns 128 keys of one key head, 32 to a wave, and
// runs over the rows of all query heads that read it, without the tiles of rows that see none of its keys.
//   Both kernels together: bf16 heads of 256, 4 x 2000 tokens, 8 heads on 4, causal 740 us (0.22 PFLOP/s of the gradient's
// five products; dV and dK are launches of their own there, which leaves one of them its accumulators in registers, and S is
// computed three times and dP twice: eight products); fp32, 4 x 2000 tokens, 8 heads of 64, causal 713 us (57 TFLOP/s of five,
// 80 of the seven that are computed).  What else keeps them from the large products' rates has not been measured: tiles pass
// through registers, and fp32 reads turned fragments an element at a time.
#pragma once
#include "masked_attention.h"

namespace ffk {

template <typename T, int DP, int RG>
struct MaskedDq {
  static constexpr int kKW = 4 / RG;
  static constexpr int kT = 32 * kKW;
  static constexpr int kKS = TileStride<T, DP>::both, kVS = TileStride<T, DP>::row;
  static constexpr int kTile = kT * (kKS + kVS) * (int)sizeof(T);
  static constexpr int kBuffers = 2 * kTile <= 152 * 1024 ? 2 : 1;
  static constexpr int kMerge = (kKW - 1) * RG * DP * 32 * 4;
  static constexpr int kBytes = kBuffers * kTile > kMerge ? kBuffers * kTile : kMerge;
  static_assert(kBytes <= 156 * 1024, "LDS of a CU");
};

template <typename T, int DP, int RG, int EXTRA>
__global__ __launch_bounds__(256) void masked_dq_kernel(MaskedAttnParams p) {
  using C = MaskedDq<T, DP, RG>;
  constexpr int KW = C::kKW;
  constexpr int kCap = EXTRA & 3;  // kNoCap, kCapLogistic or kCapTanh
  constexpr bool kBias = (EXTRA & 4) != 0;
  extern __shared__ __attribute__((aligned(16))) uint8_t pool[];
  __shared__ int window[2][4];
  __shared__ float delta_parts[4][32];
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const qw = wave / KW, kw = wave % KW;
  int const nrb = (p.R + 32 * RG - 1) / (32 * RG);
  int kh, b, hb;
  int const rb = nrb - 1 - place_of(p, kh, b, hb);
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
  int ds_lo, ds_hi;
  score_range(lo, hi, ds_lo, ds_hi);
  int const w_lo_min = wave_min_int(lo), w_hi_max = wave_max_int(hi), w_lo_max = wave_max_int(lo), w_hi_min = wave_min_int(hi);
  int const s_lo_max = summary_lo_max(lo, hi, w_lo_max);
  if (lane == 0) {
    window[0][wave] = w_lo_min;
    window[1][wave] = w_hi_max;
    if (kh == 0 && kw == 0 && row0 < p.R)
      p.summary[(int64_t)b * ((p.R + 31) / 32) + row0 / 32] = RangeSummary{w_lo_min, w_hi_max, s_lo_max, w_hi_min};
  }
  __syncthreads();
  int const lo_all = __builtin_amdgcn_readfirstlane(min(min(window[0][0], window[0][1]), min(window[0][2], window[0][3])));
  int const hi_all = __builtin_amdgcn_readfirstlane(max(max(window[1][0], window[1][1]), max(window[1][2], window[1][3])));
  int const ntiles = hi_all > lo_all ? (hi_all - lo_all + C::kT - 1) / C::kT : 0;

  int64_t const o_at = (int64_t)b * p.o_bs + (int64_t)qi * p.o_ss + (int64_t)head * p.Dv;
  T const *qp = static_cast<T const *>(p.q) + (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * p.Dq;
  T const *gp = static_cast<T const *>(p.d_o) + o_at;
  T const *op = static_cast<T const *>(p.o) + o_at;
  T const *kp = static_cast<T const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * p.Dq;
  T const *vp = static_cast<T const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * p.Dv;
  float const slope = kBias ? p.slopes[head] * p.slope_unit : 0.0f;
  int const position = p.q_offset + qi;

  Frag<T> qf[DP / 16], gf[DP / 16];
#pragma unroll
  for (int kk = 0; kk < DP / 16; kk++) {
    qf[kk] = frag_row(qp, kk * 16 + h32 * 8, p.Dq);
    gf[kk] = frag_row(gp, kk * 16 + h32 * 8, p.Dv);
  }
  // delta: a lane holds half of its row's columns (8 of every 16), lane ^ 32 the others
  float delta = 0.0f;
#pragma unroll
  for (int kk = 0; kk < DP / 16; kk++) {
    Frag<T> const of = frag_row(op, kk * 16 + h32 * 8, p.Dv);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 8; e++) delta += (float)of.v[e] * (float)gf[kk].v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) delta += of.a[e] * gf[kk].a[e] + of.b[e] * gf[kk].b[e];
    }
  }
  delta += __shfl_xor(delta, 32, 64);
  float const lse2 = p.lse[((int64_t)b * p.H + head) * p.Sq + qi] * kLog2e - p.shift;
  if (rb == nrb - 1) write_padding(p, b, kh, nrb * 32 * RG, t);

  f32x16 dq[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) dq[i][r] = 0.0f;

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
  int const koff = lane_k_off(C::kKS, lane), voff = lane_k_off(C::kVS, lane), toff = turn_off<T>(C::kKS, lane);
  float delta_sum = 0.0f;
  // all keys; DELTA: the sum of P dP alone
  auto all_tiles = [&](auto delta_tag) __attribute__((always_inline)) {
    constexpr bool DELTA = decltype(delta_tag)::value;
    if (ntiles > 0) {
      fetch(lo_all);
      stash(0);
    }
    __syncthreads();
    int cur = 0;
    for (int it = 0; it < ntiles; it++) {
      bool const more = it + 1 < ntiles;
      if (more) fetch(lo_all + (it + 1) * C::kT);
      int const kv0 = lo_all + it * C::kT + kw * 32;
      if (kv0 < w_hi_max && kv0 + 32 > w_lo_min) {
        T const *kt = k_tile(cur) + kw * 32 * C::kKS, *vt = v_tile(cur) + kw * 32 * C::kVS + voff;
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[r] = 0.0f;
          dp[r] = 0.0f;
        }
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) {
          mma(s, frag_lds(kt + koff + kk * 16), qf[kk]);
          mma(dp, frag_lds(vt + kk * 16), gf[kk]);
        }
        float ds[16];
        bool const whole = kv0 >= w_lo_max && kv0 + 32 <= w_hi_min;
        float const distance = (float)(position - (kv0 + 4 * h32));
#pragma unroll
        for (int r = 0; r < 16; r++) {
          float const y = capped<kCap>(p, s[r]);
          float x = y;
          if constexpr (kBias) x = __builtin_fmaf(-slope, fabsf(distance - (float)(8 * (r >> 2) + (r & 3))), x);
          ds[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, p.score_scale, -lse2)) * (DELTA ? dp[r] : dp[r] - delta);
          if constexpr (kCap != kNoCap && !DELTA) ds[r] *= capped_slope<kCap>(y);
        }
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            int const kv = kv0 + 8 * (r >> 2) + 4 * h32 + (r & 3);
            if (kv < ds_lo || kv >= ds_hi) ds[r] = 0.0f;
          }
        }
        if constexpr (DELTA) {
#pragma unroll
          for (int r = 0; r < 16; r++) delta_sum += ds[r];
        } else {
#pragma unroll
          for (int s2 = 0; s2 < 2; s2++) {
            Frag<T> const df = frag_acc(ds + 8 * s2, kp);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) mma(dq[i], frag_turned(kt + toff, C::kKS, s2, i * 32), df);
          }
        }
      }
      if constexpr (C::kBuffers == 2) {
        if (more) stash(cur ^ 1);
        __syncthreads();
        cur ^= 1;
      } else {
        __syncthreads();
        if (more) stash(0);
        __syncthreads();
      }
    }
  };
  if constexpr (sizeof(T) == 2) {
    if (ntiles > 0 && hi_all - lo_all <= kExactDelta) {  // uniform
      all_tiles(std::true_type{});
      delta = delta_sum + __shfl_xor(delta_sum, 32, 64);
      if constexpr (KW > 1) {
        if (lane < 32) delta_parts[wave][lane] = delta;
        __syncthreads();
        delta = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; w++) delta += delta_parts[qw * KW + w][lane & 31];
      }
    }
  }
  if (h32 == 0 && kw == 0) write_row(p, b, kh, row, lse2, delta, lo, hi, slope, position);
  all_tiles(std::false_type{});

  if constexpr (KW > 1) {
    float *const area = reinterpret_cast<float *>(pool);
    __syncthreads();
    if (kw > 0) {
      float *to = area + ((kw - 1) * RG + qw) * DP * 32;
#pragma unroll
      for (int i = 0; i < DP / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) to[(i * 16 + r) * 64 + lane] = dq[i][r];
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int w = 0; w < KW - 1; w++) {
      float const *from = area + (w * RG + qw) * DP * 32;
#pragma unroll
      for (int i = 0; i < DP / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) dq[i][r] += from[(i * 16 + r) * 64 + lane];
    }
  }
  if (row >= p.R) return;
  T *dqp = static_cast<T *>(p.dq) + (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * p.Dq;
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      int const d = i * 32 + 8 * g + 4 * h32;
      if (d < p.Dq)
        store4(dqp + d, dq[i][4 * g] * p.grad_scale, dq[i][4 * g + 1] * p.grad_scale, dq[i][4 * g + 2] * p.grad_scale, dq[i][4 * g + 3] * p.grad_scale);
    }
}

template <typename T, int DP, int KG>
struct MaskedDkdv {
  static constexpr int kKW = 4 / KG;
  static constexpr int kT = 32 * kKW;  // rows of a step
  static constexpr int kS = TileStride<T, DP>::both;
  static constexpr int kTile = 2 * kT * kS * (int)sizeof(T);  // Q and dO
  static constexpr int kBuffers = 2 * kTile <= 144 * 1024 ? 2 : 1;
  static constexpr int kMerge = (kKW - 1) * KG * DP * 32 * 4;
  static constexpr int kBytes = kBuffers * kTile > kMerge ? kBuffers * kTile : kMerge;
  static_assert(kBytes <= 154 * 1024, "LDS of a CU");
};

// KG groups of 32 keys, whose KW = 4 / KG waves take the tiles of 32 rows in turn (their sums meet in LDS at the end).
// WHAT: bit 0 dV, bit 1 dK.  Both from one launch, but where the owned K and V rows and both accumulators are more than
// a wave's registers.
template <typename T, int DP, int KG, int WHAT, int EXTRA>
__global__ __launch_bounds__(256) void masked_dkdv_kernel(MaskedAttnParams p) {
  using C = MaskedDkdv<T, DP, KG>;
  constexpr int KW = C::kKW, kT = C::kT;
  constexpr bool kDv = (WHAT & 1) != 0, kDk = (WHAT & 2) != 0;
  // bf16 past 128 columns: the accumulators, half of a lane's registers, stay in accumulation registers, so that the other
  // half holds operands read ahead
  constexpr bool kKept = sizeof(T) == 2 && DP > 128;
  constexpr int kCap = EXTRA & 3;  // kNoCap, kCapLogistic or kCapTanh
  constexpr bool kBias = (EXTRA & 4) != 0;
  extern __shared__ __attribute__((aligned(16))) uint8_t pool[];
  __shared__ __attribute__((aligned(16))) float stats[C::kBuffers][kRowFields][kT];  // integers by their bits
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const kg = wave / KW, kw = wave % KW;
  int kh, b, hb;
  int const kv0 = place_of(p, kh, b, hb) * 32 * KG;  // under a causal mask the first keys are seen by most rows
  int const wkv0 = kv0 + kg * 32, kv = wkv0 + (lane & 31);
  int const nsum = (p.R + 31) / 32, nsteps = (nsum + KW - 1) / KW;
  RangeSummary const *sums = p.summary + (int64_t)b * nsum;

  T const *kp = static_cast<T const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)min(kv, p.Skv - 1) * p.k_ss + (int64_t)kh * p.Dq;
  T const *vp = static_cast<T const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)min(kv, p.Skv - 1) * p.v_ss + (int64_t)kh * p.Dv;
  T const *qp = static_cast<T const *>(p.q) + (int64_t)b * p.q_bs;
  T const *gp = static_cast<T const *>(p.d_o) + (int64_t)b * p.o_bs;

  Frag<T> kf[DP / 16], vf[kDk ? DP / 16 : 1];
#pragma unroll
  for (int kk = 0; kk < DP / 16; kk++) {
    kf[kk] = frag_row(kp, kk * 16 + h32 * 8, p.Dq);
    if constexpr (kDk) vf[kk] = frag_row(vp, kk * 16 + h32 * 8, p.Dv);
  }
  f32x16 dk[kDk ? DP / 32 : 1], dv[kDv ? DP / 32 : 1];
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      if constexpr (kDk) dk[i][r] = 0.0f;
      if constexpr (kDv) dv[i][r] = 0.0f;
    }
  if constexpr (kKept) {
#pragma unroll
    for (int i = 0; i < DP / 32; i++) {
      if constexpr (kDk) asm volatile("" : "+a"(dk[i]));
      if constexpr (kDv) asm volatile("" : "+a"(dv[i]));
    }
  }

  auto q_tile = [&](int buf) { return reinterpret_cast<T *>(pool + buf * C::kTile); };
  auto g_tile = [&](int buf) { return q_tile(buf) + kT * C::kS; };
  // Which tiles: a lane holds the summary of one of 64, read before they are needed, so that no step waits for memory to
  // know its tile (a load behind those of the next tile's rows would wait for them too).
  RangeSummary mine;
  uint64_t wanted = 0;  // tiles with a row that sees a key of this workgroup
  int group = -1;
  auto next = [&](int step) {  // the first step at or behind `step` that has such a tile
    int tile = step * KW;
    while (tile < nsum) {
      if (tile >> 6 != group) {
        group = tile >> 6;
        int const at = group * 64 + lane;
        mine = at < nsum ? sums[at] : RangeSummary{1 << 30, 0, 1 << 30, 0};
        wanted = __builtin_amdgcn_ballot_w64(mine.lo_min < kv0 + 32 * KG && mine.hi_max > kv0);
      }
      uint64_t const left = wanted >> (tile & 63);
      if (left != 0) return (tile + __builtin_ctzll(left)) / KW;
      tile = (tile & ~63) + 64;
    }
    return nsteps;
  };
  auto summary_of = [&](int tile) {  // of the tiles that `next` looked at last
    int const at = tile & 63;
    return RangeSummary{__builtin_amdgcn_readlane(mine.lo_min, at), __builtin_amdgcn_readlane(mine.hi_max, at),
                        __builtin_amdgcn_readlane(mine.lo_max, at), __builtin_amdgcn_readlane(mine.hi_min, at)};
  };
  using Regs = TileRegs<T, DP, kT>;
  Regs tq, tg;
  int seen_lo[Regs::kN], seen_hi[Regs::kN];  // of this thread's rows: one that sees none of the keys is a row of zeros in LDS
  float field[kRowFields];                   // of row t of the step
  float const *rows = p.rows + (int64_t)hb * kRowFields * p.padded_rows;
  auto fetch = [&](int step) {
#pragma unroll
    for (int n = 0; n < Regs::kN; n++) {
      int const r = min(step * kT + (t + n * 256) / Regs::kCPR, p.padded_rows - 1);
      seen_lo[n] = __float_as_int(rows[kRowLo * (int64_t)p.padded_rows + r]);
      seen_hi[n] = __float_as_int(rows[kRowHi * (int64_t)p.padded_rows + r]);
    }
    auto offset = [&](int r, int64_t seq_stride, int D) {
      int i, g;
      row_of(p, min(step * kT + r, p.R - 1), i, g);
      return (int64_t)i * seq_stride + (int64_t)(kh * p.G + g) * D;
    };
    tq.load([&](int r) { return qp + offset(r, p.q_ss, p.Dq); }, p.Dq, t);
    tg.load([&](int r) { return gp + offset(r, p.o_ss, p.Dv); }, p.Dv, t);
    int const r = min(step * kT + min(t, kT - 1), p.padded_rows - 1);
#pragma unroll
    for (int f = 0; f < (kBias ? kRowFields : kRowSlope); f++) field[f] = rows[f * (int64_t)p.padded_rows + r];
  };
  auto stash = [&](int buf, int step) {
    auto keep = [&](int n) {
      int const r = step * kT + (t + n * 256) / Regs::kCPR;
      return r < p.R && seen_lo[n] < kv0 + 32 * KG && seen_hi[n] > kv0;
    };
    tq.store(q_tile(buf), C::kS, p.Dq, t, keep);
    tg.store(g_tile(buf), C::kS, p.Dv, t, keep);
    if (t < kT) {
#pragma unroll
      for (int f = 0; f < (kBias ? kRowFields : kRowSlope); f++)
        stats[buf][f][t] = f == kRowHi && step * kT + t >= p.R ? __int_as_float(0) : field[f];
    }
  };
  int const roff = lane_k_off(C::kS, lane), toff = turn_off<T>(C::kS, lane);
  int step = __builtin_amdgcn_readfirstlane(next(0));
  if (step < nsteps) {
    fetch(step);
    stash(0, step);
  }
  __syncthreads();
  int cur = 0;
  while (step < nsteps) {
    RangeSummary const sum = summary_of(step * KW + kw);
    int const after = __builtin_amdgcn_readfirstlane(next(step + 1));
    if (after < nsteps) fetch(after);
    if (wkv0 < p.Skv && sum.lo_min < wkv0 + 32 && sum.hi_max > wkv0) {
      T const *qt = q_tile(cur) + kw * 32 * C::kS, *gt = g_tile(cur) + kw * 32 * C::kS;
      // a field of the rows of scores 4 g .. + 3
      auto rows4 = [&](int f, int g) { return *reinterpret_cast<f32x4 const *>(&stats[cur][f][kw * 32 + 8 * g + 4 * h32]); };
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        s[r] = 0.0f;
        dp[r] = 0.0f;
      }
      if constexpr (kKept) {
        constexpr int W = kDk ? 2 : 1, N = W * DP / 16, kAhead = 4;
        Frag<T> fr[kAhead + 1];
        auto fragment = [&](int n) { return frag_lds((n % W == 0 ? qt : gt) + roff + n / W * 16); };
#pragma unroll
        for (int n = 0; n < kAhead; n++) fr[n] = fragment(n);
#pragma unroll
        for (int n = 0; n < N; n++) {
          if (n + kAhead < N) fr[(n + kAhead) % (kAhead + 1)] = fragment(n + kAhead);
          __builtin_amdgcn_sched_barrier(0);
          if (n % W == 0) mma(s, fr[n % (kAhead + 1)], kf[n / W]);
          else mma(dp, fr[n % (kAhead + 1)], vf[n / W]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++) {
          mma(s, frag_lds(qt + roff + kk * 16), kf[kk]);
          if constexpr (kDk) mma(dp, frag_lds(gt + roff + kk * 16), vf[kk]);
        }
      }
      float pv[16], ds[16];
      bool const whole = wkv0 >= sum.lo_max && wkv0 + 32 <= sum.hi_min;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        f32x4 const lse4 = rows4(kRowLse2, g);
        f32x4 delta4, slope4, position4;
        if constexpr (kDk) delta4 = rows4(kRowDelta, g);
        if constexpr (kBias) {
          slope4 = rows4(kRowSlope, g);
          position4 = rows4(kRowPosition, g);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          int const r = 4 * g + e;
          float const y = capped<kCap>(p, s[r]);
          float x = y;
          if constexpr (kBias) x = __builtin_fmaf(-slope4[e], (float)abs(__float_as_int(position4[e]) - kv), x);
          pv[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, p.score_scale, -lse4[e]));
          if constexpr (kDk) {
            ds[r] = pv[r] * (dp[r] - delta4[e]);
            if constexpr (kCap != kNoCap) ds[r] *= capped_slope<kCap>(y);
          }
        }
      }
      if (!whole) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
          f32x4 const lo4 = rows4(kRowLo, g), hi4 = rows4(kRowHi, g);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (kv < __float_as_int(lo4[e]) || kv >= __float_as_int(hi4[e])) {
              pv[4 * g + e] = 0.0f;
              if constexpr (kDk) ds[4 * g + e] = 0.0f;
            }
          }
        }
        if (sum.lo_max == 1 << 30) {  // (rows that see one key, or none)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            f32x4 const lo4 = rows4(kRowLo, g), hi4 = rows4(kRowHi, g);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              if (one_key(__float_as_int(lo4[e]), __float_as_int(hi4[e]))) {
                pv[4 * g + e] = kv == __float_as_int(lo4[e]) ? 1.0f : 0.0f;
                if constexpr (kDk) ds[4 * g + e] = 0.0f;
              }
            }
          }
        }
      }
      if constexpr (kKept) {
        // (one of the two products: WHAT is 1 or 2 past 128 columns)
        bf16x8 of[2] = {pack8(kDv ? pv : ds), pack8((kDv ? pv : ds) + 8)};
        bf16 const *from = (kDv ? gt : qt) + toff;
        constexpr int N = DP / 16, kAhead = 4;
        bf16x8 fr[kAhead + 1];
#pragma unroll
        for (int n = 0; n < kAhead; n++) fr[n] = frag_turned(from, C::kS, n / (DP / 32), n % (DP / 32) * 32).v;
        asm volatile("s_nop 3" : "+v"(of[0]), "+v"(of[1]));  // the wait states between a vector instruction and mma_kept
#pragma unroll
        for (int n = 0; n < N; n++) {
          if (n + kAhead < N) fr[(n + kAhead) % (kAhead + 1)] = frag_turned(from, C::kS, (n + kAhead) / (DP / 32), (n + kAhead) % (DP / 32) * 32).v;
          if constexpr (kDv) mma_kept(dv[n % (DP / 32)], fr[n % (kAhead + 1)], of[n / (DP / 32)]);
          else mma_kept(dk[n % (DP / 32)], fr[n % (kAhead + 1)], of[n / (DP / 32)]);
        }
      } else {
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
          if constexpr (kDv) {
            Frag<T> const pf = frag_acc(pv + 8 * s2, kp);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) mma(dv[i], frag_turned(gt + toff, C::kS, s2, i * 32), pf);
          }
          if constexpr (kDk) {
            Frag<T> const df = frag_acc(ds + 8 * s2, kp);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) mma(dk[i], frag_turned(qt + toff, C::kS, s2, i * 32), df);
          }
        }
      }
    }
    if constexpr (C::kBuffers == 2) {
      if (after < nsteps) stash(cur ^ 1, after);
      __syncthreads();
      cur ^= 1;
    } else {
      __syncthreads();
      if (after < nsteps) stash(0, after);
      __syncthreads();
    }
    step = after;
  }

  if constexpr (kKept && kDv) mma_settled(dv);
  if constexpr (kKept && kDk) mma_settled(dk);
  // the sums of the waves of a group, added up by its first, and written out: a lane owns a key
  auto finish = [&](f32x16 (&acc)[DP / 32], float factor, T *out, int D) {
    if constexpr (KW > 1) {
      float *const area = reinterpret_cast<float *>(pool);
      __syncthreads();
      if (kw > 0) {
        float *to = area + ((kw - 1) * KG + kg) * DP * 32;
#pragma unroll
        for (int i = 0; i < DP / 32; i++)
#pragma unroll
          for (int r = 0; r < 16; r++) to[(i * 16 + r) * 64 + lane] = acc[i][r];
      }
      __syncthreads();
      if (kw == 0) {
#pragma unroll
        for (int w = 0; w < KW - 1; w++) {
          float const *from = area + (w * KG + kg) * DP * 32;
#pragma unroll
          for (int i = 0; i < DP / 32; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][r] += from[(i * 16 + r) * 64 + lane];
        }
      }
    }
    if (kw == 0 && kv < p.Skv) {
#pragma unroll
      for (int i = 0; i < DP / 32; i++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          int const d = i * 32 + 8 * g + 4 * h32;
          if (d < D) store4(out + d, acc[i][4 * g] * factor, acc[i][4 * g + 1] * factor, acc[i][4 * g + 2] * factor, acc[i][4 * g + 3] * factor);
        }
    }
  };
  if constexpr (kDk) finish(dk, p.grad_scale, static_cast<T *>(p.dk) + (int64_t)b * p.k_bs + (int64_t)kv * p.k_ss + (int64_t)kh * p.Dq, p.Dq);
  if constexpr (kDv) finish(dv, 1.0f, static_cast<T *>(p.dv) + (int64_t)b * p.v_bs + (int64_t)kv * p.v_ss + (int64_t)kh * p.Dv, p.Dv);
}

template <typename T, int DP, int RG, int EXTRA>
static hipError_t masked_dq_launch_as(hipStream_t st, MaskedAttnParams const &p) {
  static LdsOptIn opt_in;
  using C = MaskedDq<T, DP, RG>;
  auto kernel = &masked_dq_kernel<T, DP, RG, EXTRA>;
  hipError_t e = opt_in.ensure(reinterpret_cast<void const *>(kernel), C::kBytes);
  if (e != hipSuccess) return e;
  int64_t const grid = ceil_div(p.R, 32 * RG) * p.KH * p.B;
  kernel<<<dim3((unsigned)grid), 256, C::kBytes, st>>>(p);
  return hipGetLastError();
}

template <typename T, int DP, int KG, int WHAT, int EXTRA>
static hipError_t masked_dkdv_launch_as(hipStream_t st, MaskedAttnParams const &p) {
  static LdsOptIn opt_in;
  using C = MaskedDkdv<T, DP, KG>;
  auto kernel = &masked_dkdv_kernel<T, DP, KG, WHAT, EXTRA>;
  hipError_t e = opt_in.ensure(reinterpret_cast<void const *>(kernel), C::kBytes);
  if (e != hipSuccess) return e;
  int64_t const grid = ceil_div(p.Skv, 32 * KG) * p.KH * p.B;
  kernel<<<dim3((unsigned)grid), 256, C::kBytes, st>>>(p);
  return hipGetLastError();
}

template <typename T, int DP, int RG>
static hipError_t masked_dq_launch(hipStream_t st, MaskedAttnParams const &p) {
  return masked_by_score<T>(p, [&](auto extra) { return masked_dq_launch_as<T, DP, RG, decltype(extra)::value>(st, p); });
}

template <typename T, int DP, int KG, int WHAT>
static hipError_t masked_dkdv_launch(hipStream_t st, MaskedAttnParams const &p) {
  return masked_by_score<T>(p, [&](auto extra) { return masked_dkdv_launch_as<T, DP, KG, WHAT, decltype(extra)::value>(st, p); });
}

}  // namespace ffk
