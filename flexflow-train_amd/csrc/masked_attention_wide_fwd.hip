// Masked attention, forward for bf16 heads of 64 and 128 with 64 rows to a wave (see masked_attention.h for the
// mathematics and layouts).
//
// One workgroup takes 256 rows of one key head, one wave runs on a SIMD and owns 64 of them as two halves of 32.  For a
// tile of 64 keys both halves use the same K and V fragments, and the wave overlaps matrix and vector work itself:
//   phase 1   S_0 = K Q_0^T                     phase 2   S_1 = K Q_1^T   next to the softmax of S_0
//   phase 3   O_0 += V^T P_0 next to the softmax of S_1     phase 4   O_1 += V^T P_1
// The softmax of a half is cut into units that sit behind the MFMAs of phases 2 and 3, fenced against the scheduler.
// K and V arrive by direct loads, one tile ahead, as they lie in memory but for a permutation of the 16-byte chunks of a
// row on the fetching side, which keeps the reads free of bank conflicts.
//   The loop runs over the union of the rows' ranges.  A wave passes over a tile that none of its rows sees, and ranges
// are compared element by element only where a tile is not seen whole by all of its rows.
#include "masked_attention.h"
#include "lds_dma.h"

namespace ffk {

template <int D>
struct WideFwd {
  static constexpr int kRows = 256, kKeys = 64;
  static constexpr int kCPR = D / 8;
  static constexpr int kLoads = kKeys * kCPR / 256;
  static constexpr int kRowsPerLoad = 256 / kCPR;
  static constexpr int kTile = kKeys * D;
  __device__ static int kswz(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
  __device__ static int vswz(int row) { return D == 128 ? (row & 3) : ((row >> 1) & 1); }
  static_assert(D == 64 || D == 128, "permutations are written for these two");
};

// Online softmax of one half (32 rows x 64 keys: two score blocks, this lane's column) in 16 units.
//   plain scores:     units 0..3 the maximum of 8 raw scores each; unit 4 the new reference point; units 5..15 three
//                     exponentials each (the last two), summed as they come
//   capped or biased: units 0..7 turn 4 raw scores each into scores in powers of two, masked where the tile is not
//                     seen whole, and take their maximum; unit 8 the reference point; units 9..15 five exponentials each
// The reference point of the exponentials moves only when the maximum has grown by more than kLazy (in powers of two):
// until then probabilities may exceed 1 (by at most 2^kLazy, harmless in 32-bit sums and in bf16's range) and the sums keep
// their scale, which saves the rescaling of the accumulators in nearly every tile.
template <bool CAP, bool BIAS>
struct MaskedSoftmax {
  static constexpr float kLazy = 8.0f;
  static constexpr bool kExtra = CAP || BIAS;
  static constexpr int kReference = kExtra ? 8 : 4, kPer = kExtra ? 5 : 3;
  float mx, m_use, m_new, alpha, sum;
  float pv[2][16];
  template <int UNIT>
  __device__ __forceinline__ void unit(MaskedAttnParams const &p, f32x16 (&s)[2], float m_run, bool edge, int kv_first, int lo, int hi,
                                       float slope2, int position) {
    if constexpr (UNIT < kReference) {
      if constexpr (kExtra) {
        constexpr int j = UNIT / 4, first = (UNIT % 4) * 4;
#pragma unroll
        for (int r = first; r < first + 4; r++) {
          float x = CAP ? p.cap_out * cap_tanh<bf16>(p, s[j][r]) : s[j][r] * p.scale_log2;
          // the keys of an accumulator: 8 (r / 4) + r % 4 behind the lane's first
          if constexpr (BIAS) x = __builtin_fmaf(-slope2, (float)abs(position - (kv_first + j * 32 + 8 * (r >> 2) + (r & 3))), x);
          s[j][r] = x;
        }
        if (edge) {
#pragma unroll
          for (int r = first; r < first + 4; r++) {
            int const kv = kv_first + j * 32 + 8 * (r >> 2) + (r & 3);
            if (kv < lo || kv >= hi) s[j][r] = -INFINITY;
          }
        }
        float const a = fmaxf(fmaxf(s[j][first], s[j][first + 1]), s[j][first + 2]);
        mx = UNIT == 0 ? fmaxf(a, s[j][first + 3]) : fmaxf(fmaxf(mx, a), s[j][first + 3]);
      } else {
#pragma unroll
        for (int r = 4 * UNIT; r < 4 * UNIT + 4; r++) mx = r == 0 ? fmaxf(s[0][r], s[1][r]) : fmaxf(fmaxf(mx, s[0][r]), s[1][r]);
      }
      pin_here(mx);
    } else if constexpr (UNIT == kReference) {
      float const m = kExtra ? max_across_halves(mx) : max_across_halves(mx) * p.scale_log2;  // (the scale is positive)
      m_new = m > m_run + kLazy ? m : m_run;
      m_use = m_new == -INFINITY ? 0.0f : m_new;  // nothing seen yet: every exponential is 0
      alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_use);
      sum = 0.0f;
      pin_here(m_use);
      pin_here(alpha);
    } else {
      constexpr int first = (UNIT - kReference - 1) * kPer;
      constexpr int last = first + kPer < 32 ? first + kPer : 32;
#pragma unroll
      for (int e = first; e < last; e++) {
        float const x = kExtra ? s[e / 16][e % 16] - m_use : __builtin_fmaf(s[e / 16][e % 16], p.scale_log2, -m_use);
        pv[e / 16][e % 16] = __builtin_amdgcn_exp2f(x);
        sum += pv[e / 16][e % 16];
        pin_here(pv[e / 16][e % 16]);
      }
      pin_here(sum);
    }
  }
  __device__ __forceinline__ void finish(bf16x8 (&pf)[4], float &m_run, float &l_part) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      pf[2 * j] = pack8(pv[j]);
      pf[2 * j + 1] = pack8(pv[j] + 8);
    }
    l_part = l_part * alpha + sum;
    m_run = m_new;
  }
};

template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) void masked_fwd_wide_kernel(MaskedAttnParams p) {
  using C = WideFwd<D>;
  using Softmax = MaskedSoftmax<CAP, BIAS>;
  __shared__ __attribute__((aligned(1024))) bf16 Ks[2][C::kTile];
  __shared__ __attribute__((aligned(1024))) bf16 Vs[2][C::kTile];
  __shared__ int window[2][4];
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const nrb = (p.R + C::kRows - 1) / C::kRows;
  int const hb = blockIdx.x % (p.KH * p.B);
  int const rb = nrb - 1 - blockIdx.x / (p.KH * p.B);  // under a causal mask the heaviest rows go first
  int const kh = hb % p.KH, b = hb / p.KH;
  int const row0 = rb * C::kRows + wave * 64;
  int row[2], qi[2], head[2], lo[2], hi[2], position[2];
  float slope2[2] = {0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < 2; c++) {
    int g;
    row[c] = row0 + c * 32 + (lane & 31);
    row_of(p, min(row[c], p.R - 1), qi[c], g);
    head[c] = kh * p.G + g;
    position[c] = p.q_offset + qi[c];
    row_range(p, b, qi[c], lo[c], hi[c]);
    if (row[c] >= p.R) {
      lo[c] = 1 << 30;
      hi[c] = 0;
    }
    if constexpr (BIAS) slope2[c] = p.slopes[head[c]] * kLog2e;
  }
  int const w_lo_min = wave_min_int(min(lo[0], lo[1])), w_hi_max = wave_max_int(max(hi[0], hi[1]));
  // rows that do not exist narrow nothing
  int const w_lo_max = wave_max_int(max(row[0] < p.R ? lo[0] : 0, row[1] < p.R ? lo[1] : 0));
  int const w_hi_min = wave_min_int(min(row[0] < p.R ? hi[0] : 1 << 30, row[1] < p.R ? hi[1] : 1 << 30));
  if (lane == 0) {
    window[0][wave] = w_lo_min;
    window[1][wave] = w_hi_max;
  }
  __syncthreads();
  int const lo_all = __builtin_amdgcn_readfirstlane(min(min(window[0][0], window[0][1]), min(window[0][2], window[0][3])));
  int const hi_all = __builtin_amdgcn_readfirstlane(max(max(window[1][0], window[1][1]), max(window[1][2], window[1][3])));
  int const ntiles = hi_all > lo_all ? (hi_all - lo_all + C::kKeys - 1) / C::kKeys : 0;
  bf16 const *kp = uniform_pointer(static_cast<bf16 const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * D);
  bf16 const *vp = uniform_pointer(static_cast<bf16 const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * D);

  // Q as the B operand of S^T = K Q^T: column = row, k = d
  bf16x8 qf[2][D / 16];
#pragma unroll
  for (int c = 0; c < 2; c++) {
    bf16 const *qp = static_cast<bf16 const *>(p.q) + (int64_t)b * p.q_bs + (int64_t)qi[c] * p.q_ss + (int64_t)head[c] * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++) qf[c][kk] = *reinterpret_cast<bf16x8 const *>(qp + kk * 16 + h32 * 8);
  }

  // Direct loads: thread slot c (of 256 a load) writes LDS chunk c of the load's 4 KB and fetches the chunk that the
  // permutation puts there.
  int const slot_row = t / C::kCPR, slot_pc = t % C::kCPR;
  int const k_lc = slot_pc ^ C::kswz(slot_row);
  int const v_lc = ((((slot_pc >> 2) ^ C::vswz(slot_row)) << 2) | (slot_pc & 3));
  unsigned const ks_addr = lds_address_of(&Ks[0][0]), vs_addr = lds_address_of(&Vs[0][0]);
  unsigned k_voff[C::kLoads], v_voff[C::kLoads];  // of a tile that lies wholly below hi_all
#pragma unroll
  for (int i = 0; i < C::kLoads; i++) {
    k_voff[i] = (unsigned)((slot_row + i * C::kRowsPerLoad) * p.k_ss + k_lc * 8) * 2u;
    v_voff[i] = (unsigned)((slot_row + i * C::kRowsPerLoad) * p.v_ss + v_lc * 8) * 2u;
  }
  auto issue_tile = [&](int kv0, int buf) {
    i32x4 const k_rsrc = buffer_resource(kp + (int64_t)kv0 * p.k_ss);
    i32x4 const v_rsrc = buffer_resource(vp + (int64_t)kv0 * p.v_ss);
    unsigned const k_dst = ks_addr + (unsigned)(buf * C::kTile * 2 + wave * 1024);
    unsigned const v_dst = vs_addr + (unsigned)(buf * C::kTile * 2 + wave * 1024);
    if (kv0 + C::kKeys > hi_all) {  // uniform
      // keys past the last one that is seen repeat it: what lies there is not read
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        int const r = min(slot_row + i * C::kRowsPerLoad, hi_all - 1 - kv0);
        lds_dma16(k_rsrc, (unsigned)(r * p.k_ss + k_lc * 8) * 2u, 0u, k_dst + (unsigned)(i * 4096));
      }
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        int const r = min(slot_row + i * C::kRowsPerLoad, hi_all - 1 - kv0);
        lds_dma16(v_rsrc, (unsigned)(r * p.v_ss + v_lc * 8) * 2u, 0u, v_dst + (unsigned)(i * 4096));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) lds_dma16(k_rsrc, k_voff[i], 0u, k_dst + (unsigned)(i * 4096));
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) lds_dma16(v_rsrc, v_voff[i], 0u, v_dst + (unsigned)(i * 4096));
    }
  };

  f32x16 oacc[2][D / 32];
#pragma unroll
  for (int c = 0; c < 2; c++)
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) oacc[c][i][r] = 0.0f;
  float m_run[2] = {-INFINITY, -INFINITY};
  float l_part[2] = {0.0f, 0.0f};  // this lane's 16 of every 32 keys; the two lane halves meet at the end

  // K fragment (key block j, d step kk): row j*32 + l%32, chunk (2 kk + l/32) ^ kswz(row)
  int k_off[D / 16];
#pragma unroll
  for (int kk = 0; kk < D / 16; kk++) k_off[kk] = (lane & 31) * D + (((2 * kk + h32) ^ C::kswz(lane & 31)) << 3);
  // V fragment (d block i): rows 4 (l/32) + (l%16)/4 (+ 8) of a 16-row step, 4 columns at 16 ((l/16)%2) + 4 (l%4)
  int v_off[D / 32];
  {
    int const i16 = lane & 15, lr = 4 * h32 + (i16 >> 2);
#pragma unroll
    for (int i = 0; i < D / 32; i++) v_off[i] = lr * D + ((i ^ C::vswz(lr)) << 5) + ((lane >> 4) & 1) * 16 + (i16 & 3) * 4;
  }
  auto k_frag = [&](bf16 const *tile, int j, int kk) -> bf16x8 { return *reinterpret_cast<bf16x8 const *>(tile + k_off[kk] + j * 32 * D); };
  auto v_frag = [&](bf16 const *tile, int js, int i) -> bf16x8 {
    bf16 const *q = tile + v_off[i] + js * 16 * D;  // js = 2 (key block) + step
    union {
      s16x4 h2[2];
      bf16x8 v;
    } u;
    u.h2[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(q));
    u.h2[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(q + 8 * D));
    return u.v;
  };
  if (ntiles > 0) issue_tile(lo_all, 0);
  wait_all_vmem_known_to_compiler();  // the Q fragments too: no wait for them inside the loop
  __syncthreads();
  auto tile_step = [&](int it, auto buffer_tag) __attribute__((always_inline)) {
    constexpr int cur = decltype(buffer_tag)::value;
    int const kv0 = lo_all + it * C::kKeys;
    if (it + 1 < ntiles) issue_tile(kv0 + C::kKeys, cur ^ 1);
    if (kv0 < w_hi_max && kv0 + C::kKeys > w_lo_min) {
      bf16 const *kt = Ks[cur], *vt = Vs[cur];
      bool const edge = kv0 < w_lo_max || kv0 + C::kKeys > w_hi_min;
      int const kv_first = kv0 + 4 * h32;
      auto mask = [&](f32x16 (&s)[2], int c) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            int const kv = kv_first + j * 32 + 8 * (r >> 2) + (r & 3);
            if (kv < lo[c] || kv >= hi[c]) s[j][r] = -INFINITY;
          }
      };
      auto rescale = [&](int c, float alpha) {
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
          asm volatile("" ::: "memory");  // keeps the multiplications under the branch
#pragma unroll
          for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) oacc[c][i][r] *= alpha;
        }
      };

      // ---- phase 1 ----
      bf16x8 kf[2][D / 16];
#pragma unroll
      for (int kk = 0; kk < D / 16; kk++)
#pragma unroll
        for (int j = 0; j < 2; j++) kf[j][kk] = k_frag(kt, j, kk);
      f32x16 s0[2], s1[2];
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s0[j][r] = 0.0f;
          s1[j][r] = 0.0f;
        }
      constexpr int NM = D / 8;     // MFMAs of a phase
      constexpr int UPM = 16 / NM;  // softmax units behind each
      static_for<0, NM>([&](auto mc) {
        constexpr int m = decltype(mc)::value;
        constexpr int kk = m / 2, j = m % 2;
        __builtin_amdgcn_sched_barrier(0);
        s0[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j][kk], qf[0][kk], s0[j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      });
      __builtin_amdgcn_sched_barrier(0);
      if (!Softmax::kExtra && edge) mask(s0, 0);

      // ---- phase 2 ----
      bf16x8 pf0[4], pf1[4];
      Softmax sm;
      static_for<0, NM>([&](auto mc) {
        constexpr int m = decltype(mc)::value;
        constexpr int kk = m / 2, j = m % 2;
        __builtin_amdgcn_sched_barrier(0);
        s1[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j][kk], qf[1][kk], s1[j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        static_for<0, UPM>([&](auto uc) {
          sm.template unit<m * UPM + decltype(uc)::value>(p, s0, m_run[0], edge, kv_first, lo[0], hi[0], slope2[0], position[0]);
        });
      });
      __builtin_amdgcn_sched_barrier(0);
      float const alpha0 = sm.alpha;
      sm.finish(pf0, m_run[0], l_part[0]);
      rescale(0, alpha0);
      if (!Softmax::kExtra && edge) mask(s1, 1);

      // ---- phase 3: a fragment is read kAhead MFMAs ahead of its use ----
      constexpr int kAhead = 3;
      bf16x8 vf[D / 32][4];
#pragma unroll
      for (int m = 0; m < kAhead; m++) vf[m % (D / 32)][m / (D / 32)] = v_frag(vt, m / (D / 32), m % (D / 32));
      static_for<0, NM>([&](auto mc) {
        constexpr int m = decltype(mc)::value;
        constexpr int js = m / (D / 32), i = m % (D / 32);
        __builtin_amdgcn_sched_barrier(0);
        oacc[0][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i][js], pf0[js], oacc[0][i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (m + kAhead < NM) {
          constexpr int js1 = (m + kAhead) / (D / 32), i1 = (m + kAhead) % (D / 32);
          vf[i1][js1] = v_frag(vt, js1, i1);
        }
        static_for<0, UPM>([&](auto uc) {
          sm.template unit<m * UPM + decltype(uc)::value>(p, s1, m_run[1], edge, kv_first, lo[1], hi[1], slope2[1], position[1]);
        });
      });
      __builtin_amdgcn_sched_barrier(0);
      float const alpha1 = sm.alpha;
      sm.finish(pf1, m_run[1], l_part[1]);
      rescale(1, alpha1);

      // ---- phase 4 ----
#pragma unroll
      for (int js = 0; js < 4; js++)
#pragma unroll
        for (int i = 0; i < D / 32; i++)
          oacc[1][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i][js], pf1[js], oacc[1][i], 0, 0, 0);
    }
    wait_vmcnt<0>();  // this wave's part of the next tile has landed
    __syncthreads();
  };
  for (int it = 0; it < ntiles; it += 2) {
    tile_step(it, std::integral_constant<int, 0>{});
    if (it + 1 < ntiles) tile_step(it + 1, std::integral_constant<int, 1>{});
  }

#pragma unroll
  for (int c = 0; c < 2; c++) {
    float const l = l_part[c] + __shfl_xor(l_part[c], 32, 64);
    if (row[c] < p.R) {
      float const inv = l == 0.0f ? 0.0f : 1.0f / l;
      bf16 *op = static_cast<bf16 *>(p.o) + (int64_t)b * p.o_bs + (int64_t)qi[c] * p.o_ss + (int64_t)head[c] * D;
#pragma unroll
      for (int i = 0; i < D / 32; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
          store4(op + i * 32 + 8 * g + 4 * h32, oacc[c][i][4 * g] * inv, oacc[c][i][4 * g + 1] * inv, oacc[c][i][4 * g + 2] * inv,
                 oacc[c][i][4 * g + 3] * inv);
      if (h32 == 0 && p.lse != nullptr)
        p.lse[((int64_t)b * p.H + head[c]) * p.Sq + qi[c]] = l == 0.0f ? -INFINITY : (m_run[c] + __log2f(l)) * kLn2;
    }
  }
}

template <int D>
static void launch(hipStream_t st, MaskedAttnParams const &p) {
  dim3 const grid((unsigned)(ceil_div(p.R, WideFwd<D>::kRows) * p.KH * p.B));
  bool const cap = p.cap_out != 0.0f, bias = p.slopes != nullptr;
  if (cap && bias) masked_fwd_wide_kernel<D, true, true><<<grid, 256, 0, st>>>(p);
  else if (cap) masked_fwd_wide_kernel<D, true, false><<<grid, 256, 0, st>>>(p);
  else if (bias) masked_fwd_wide_kernel<D, false, true><<<grid, 256, 0, st>>>(p);
  else masked_fwd_wide_kernel<D, false, false><<<grid, 256, 0, st>>>(p);
}

hipError_t masked_attention_fwd_wide(hipStream_t st, MaskedAttnParams const &p) {
  if (p.Dq == 64) launch<64>(st, p);
  else launch<128>(st, p);
  return hipGetLastError();
}

}  // namespace ffk
