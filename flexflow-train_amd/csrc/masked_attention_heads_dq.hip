// Masked attention, dQ for bf16 heads up to 128 (see masked_attention.h for the mathematics and layouts).
//
// One workgroup owns 128 rows of one key head, 32 to a wave, whose Q and dO rows are MFMA operands in registers; two
// workgroups run on a CU, so that the vector work of one covers the matrix work of the other.  Keys and values come in
// tiles of 64, two halves of 32, by direct loads one tile ahead, and lie in LDS as in memory but for a permutation of the
// 16-byte chunks of a row that keeps both ways of reading them free of bank conflicts (that of the dK/dV kernel).  Like
// the general kernel it leaves delta, the log-sum-exp and the ranges of its rows in memory for the dK/dV kernel, and
// summaries of the ranges.
//   Bound by the issue of vector instructions: 8192 tokens, 16 heads of 128, causal, biased 420 us (0.98 PFLOP/s with
// its three products); 4 x 4096 tokens in 3 documents, 32 heads of 128 on 8, causal, capped 490 us; 8 x 512 tokens in
// 4 documents, 16 heads of 64 21 us.
#include "masked_attention_heads.h"

namespace ffk {

template <int D>
struct HeadsDq {
  static constexpr int kKeys = 64;
  static constexpr int kCPR = D / 8;
  static constexpr int kLoads = kKeys * kCPR / 256;
  static constexpr int kRowsPerLoad = 256 / kCPR;
  static constexpr int kTile = kKeys * D;
  __device__ static int swz(int row) {
    return D == 128 ? (((row & 3) << 2) | ((row >> 2) & 3)) : ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
  }
  static_assert(D == 64 || D == 128, "permutations are written for these two");
};

template <int D, int U, bool PAD, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void masked_dq_heads_kernel(MaskedAttnParams p) {
  using C = HeadsDq<D>;
  __shared__ __attribute__((aligned(1024))) bf16 Ks[2][C::kTile];
  __shared__ __attribute__((aligned(1024))) bf16 Vs[2][C::kTile];
  __shared__ int window[2][4];
  int const dim_qk = PAD ? p.Dq : D, dim_v = PAD ? p.Dv : D;  // the heads themselves
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const nrb = (p.R + 127) / 128;
  int kh, b, hb;
  int const rb = nrb - 1 - place_of(p, kh, b, hb);
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
  int ds_lo, ds_hi;
  score_range(lo, hi, ds_lo, ds_hi);
  int64_t const q_at = (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * dim_qk;
  int64_t const o_at = (int64_t)b * p.o_bs + (int64_t)qi * p.o_ss + (int64_t)head * dim_v;
  bf16 const *qp = static_cast<bf16 const *>(p.q) + q_at, *gp = static_cast<bf16 const *>(p.d_o) + o_at;
  bf16 const *op = static_cast<bf16 const *>(p.o) + o_at;
  bf16 const *kp = uniform_pointer(static_cast<bf16 const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * dim_qk);
  bf16 const *vp = uniform_pointer(static_cast<bf16 const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * dim_v);
  bf16x8 qf[U / 16], gf[U / 16];
  float part = 0.0f;
#pragma unroll
  for (int kk = 0; kk < U / 16; kk++) {
    qf[kk] = head_chunk<PAD>(qp, kk * 16 + h32 * 8, dim_qk);
    gf[kk] = head_chunk<PAD>(gp, kk * 16 + h32 * 8, dim_v);
    bf16x8 const of = head_chunk<PAD>(op, kk * 16 + h32 * 8, dim_v);
#pragma unroll
    for (int e = 0; e < 8; e++) part += (float)of[e] * (float)gf[kk][e];
  }
  float delta = part + __shfl_xor(part, 32, 64);
  float const lse2 = p.lse[((int64_t)b * p.H + head) * p.Sq + qi] * kLog2e - p.shift;
  float slope = 0.0f;
  if constexpr (BIAS) slope = p.slopes[head] * p.slope_unit;
  int const position = p.q_offset + qi;

  int const w_lo_min = wave_min_int(lo), w_hi_max = wave_max_int(hi), w_lo_max = wave_max_int(lo), w_hi_min = wave_min_int(hi);
  int const s_lo_max = summary_lo_max(lo, hi, w_lo_max);
  if (lane == 0) {
    window[0][wave] = w_lo_min;
    window[1][wave] = w_hi_max;
    if (kh == 0 && row0 < p.R)
      p.summary[(int64_t)b * ((p.R + 31) / 32) + row0 / 32] = RangeSummary{w_lo_min, w_hi_max, s_lo_max, w_hi_min};
  }
  __syncthreads();
  int const lo_all = __builtin_amdgcn_readfirstlane(min(min(window[0][0], window[0][1]), min(window[0][2], window[0][3])));
  int const hi_all = __builtin_amdgcn_readfirstlane(max(max(window[1][0], window[1][1]), max(window[1][2], window[1][3])));
  int const ntiles = hi_all > lo_all ? (hi_all - lo_all + C::kKeys - 1) / C::kKeys : 0;

  f32x16 dq[U / 32];
#pragma unroll
  for (int i = 0; i < U / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) dq[i][r] = 0.0f;

  // Direct loads: thread slot c (of 256 a load) writes LDS chunk c of the load's 4 KB and fetches the chunk that the
  // permutation puts there.
  int const slot_row = t / C::kCPR, slot_lc = (t % C::kCPR) ^ C::swz(t / C::kCPR);
  unsigned const ks_addr = lds_address_of(&Ks[0][0]), vs_addr = lds_address_of(&Vs[0][0]);
  unsigned k_voff[C::kLoads], v_voff[C::kLoads];  // of a tile that lies wholly below hi_all
#pragma unroll
  for (int i = 0; i < C::kLoads; i++) {
    k_voff[i] = tile_offset<PAD>((slot_row + i * C::kRowsPerLoad) * p.k_ss, slot_lc * 8, dim_qk);
    v_voff[i] = tile_offset<PAD>((slot_row + i * C::kRowsPerLoad) * p.v_ss, slot_lc * 8, dim_v);
  }
  auto issue_tile = [&](int kv0, int buf) {
    i32x4 const k_rsrc = tile_resource<PAD>(kp + (int64_t)kv0 * p.k_ss);
    i32x4 const v_rsrc = tile_resource<PAD>(vp + (int64_t)kv0 * p.v_ss);
    unsigned const k_dst = ks_addr + (unsigned)(buf * C::kTile * 2 + wave * 1024);
    unsigned const v_dst = vs_addr + (unsigned)(buf * C::kTile * 2 + wave * 1024);
    if (kv0 + C::kKeys > hi_all) {  // uniform
      // keys past the last one that is seen repeat it: what lies there is not read
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        int const r = min(slot_row + i * C::kRowsPerLoad, hi_all - 1 - kv0);
        lds_dma16(k_rsrc, tile_offset<PAD>(r * p.k_ss, slot_lc * 8, dim_qk), 0u, k_dst + (unsigned)(i * 4096));
        lds_dma16(v_rsrc, tile_offset<PAD>(r * p.v_ss, slot_lc * 8, dim_v), 0u, v_dst + (unsigned)(i * 4096));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        lds_dma16(k_rsrc, k_voff[i], 0u, k_dst + (unsigned)(i * 4096));
        lds_dma16(v_rsrc, v_voff[i], 0u, v_dst + (unsigned)(i * 4096));
      }
    }
  };
  // Per-lane LDS offsets (in elements) of the two ways a tile is read (32 rows from its first row on).
  int row_off[U / 16], tr_off[U / 32][2];
  {
    int const r = lane & 31;
#pragma unroll
    for (int kk = 0; kk < U / 16; kk++) row_off[kk] = r * D + (((2 * kk + h32) ^ C::swz(r)) << 3);
    int const i16 = lane & 15, q = i16 >> 2, bb = (lane >> 4) & 1, c = i16 & 3;
#pragma unroll
    for (int i = 0; i < U / 32; i++)
#pragma unroll
      for (int sec = 0; sec < 2; sec++) {
        int const r2 = 8 * sec + 4 * h32 + q, chunk = 4 * i + 2 * bb + (c >> 1);
        tr_off[i][sec] = r2 * D + ((chunk ^ C::swz(r2)) << 3) + 4 * (c & 1);
      }
  }
  auto rows = [&](bf16 const *tile, int kk) -> bf16x8 { return *reinterpret_cast<bf16x8 const *>(tile + row_off[kk]); };
  auto turned = [&](bf16 const *tile, int s, int i) -> bf16x8 {
    union {
      s16x4 h2[2];
      bf16x8 v;
    } u;
    u.h2[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tile + tr_off[i][0] + 16 * s * D));
    u.h2[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tile + tr_off[i][1] + 16 * s * D));
    return u.v;
  };
  if (ntiles > 0) issue_tile(lo_all, 0);
  wait_all_vmem_known_to_compiler();
  __syncthreads();
  // 32 keys: S^T = K Q^T, dP^T = V dO^T (rows = keys, column = row), dS, dQ^T += K^T dS^T
  bool const exact = ntiles > 0 && ntiles * C::kKeys <= kExactDelta;  // uniform
  // A first pass over the keys then sums P dP; what it leaves in the accumulators is cleared.  (One body for both passes: a
  // second one, or a way around its products, takes registers that are not there.)
  bool first_pass = exact;
  if (exact) {
    part = 0.0f;
    delta = 0.0f;
  }
  auto half_work = [&](int kv0, bf16 const *kt, bf16 const *vt) __attribute__((always_inline)) {
    f32x16 s, dp;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      s[r] = 0.0f;
      dp[r] = 0.0f;
    }
#pragma unroll
    for (int kk = 0; kk < U / 16; kk++) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rows(kt, kk), qf[kk], s, 0, 0, 0);
      dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rows(vt, kk), gf[kk], dp, 0, 0, 0);
    }
    int const kv_first = kv0 + 4 * h32;
    float const distance = (float)(position - kv_first);
    float ds[16], y[16];
#pragma unroll
    for (int r = 0; r < 16; r++) {
      y[r] = capped<CAP ? kCapLogistic : kNoCap>(p, s[r]);
      float x = y[r];
      if constexpr (BIAS) x = __builtin_fmaf(-slope, fabsf(distance - (float)(8 * (r >> 2) + (r & 3))), x);
      ds[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, p.score_scale, -lse2)) * (dp[r] - delta);
    }
    if (first_pass) {  // uniform
      int const from = ds_lo - kv_first, to = ds_hi - kv_first;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        int const kv = 8 * (r >> 2) + (r & 3);
        part += kv < from || kv >= to ? 0.0f : ds[r];
      }
    }
    if constexpr (CAP) {
#pragma unroll
      for (int r = 0; r < 16; r++) ds[r] *= capped_slope<kCapLogistic>(y[r]);
    }
    if (kv0 < w_lo_max || kv0 + 32 > w_hi_min) {
      int const from = ds_lo - kv_first, to = ds_hi - kv_first;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        int const kv = 8 * (r >> 2) + (r & 3);
        ds[r] = kv < from || kv >= to ? 0.0f : ds[r];
      }
    }
    bf16x8 db[2] = {pack8(ds), pack8(ds + 8)};
    bf16x8 tf[4];  // a fragment is read three MFMAs ahead of its use
#pragma unroll
    for (int n = 0; n < 3; n++) tf[n] = turned(kt, n / (U / 32), n % (U / 32));
#pragma unroll
    for (int n = 0; n < U / 16; n++) {
      if (n + 3 < U / 16) tf[(n + 3) % 4] = turned(kt, (n + 3) / (U / 32), (n + 3) % (U / 32));
      dq[n % (U / 32)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tf[n % 4], db[n / (U / 32)], dq[n % (U / 32)], 0, 0, 0);
    }
  };
  auto tile_step = [&](int it, auto buffer_tag) __attribute__((always_inline)) {
    constexpr int cur = decltype(buffer_tag)::value;
    int const kv0 = lo_all + it * C::kKeys;
    // behind the last tile of the first pass the first one again
    bool const more = it + 1 < ntiles;
    if (more || first_pass) issue_tile(more ? kv0 + C::kKeys : lo_all, cur ^ 1);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if (kv0 + 32 * h < w_hi_max && kv0 + 32 * h + 32 > w_lo_min) half_work(kv0 + 32 * h, Ks[cur] + h * 32 * D, Vs[cur] + h * 32 * D);
    }
    wait_vmcnt<0>();  // this wave's part of the next tile has landed
    __syncthreads();
    if (!more && first_pass) {
      first_pass = false;
      delta = part + __shfl_xor(part, 32, 64);
#pragma unroll
      for (int i = 0; i < U / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) dq[i][r] = 0.0f;
    }
  };
  // two passes over the keys are one run of tiles, of which the second half begins again
  int const steps = exact ? 2 * ntiles : ntiles;
  for (int n = 0; n < steps; n += 2) {
    tile_step(n < ntiles ? n : n - ntiles, std::integral_constant<int, 0>{});
    if (n + 1 < steps) tile_step(n + 1 < ntiles ? n + 1 : n + 1 - ntiles, std::integral_constant<int, 1>{});
  }
  if (h32 == 0) write_row(p, b, kh, row, lse2, delta, lo, hi, slope, position);
  if (row < p.R) {
    bf16 *dqp = static_cast<bf16 *>(p.dq) + q_at;
#pragma unroll
    for (int i = 0; i < U / 32; i++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        if (!PAD || i * 32 + 8 * g + 4 * h32 < dim_qk)
          store4(dqp + i * 32 + 8 * g + 4 * h32, dq[i][4 * g] * p.grad_scale, dq[i][4 * g + 1] * p.grad_scale, dq[i][4 * g + 2] * p.grad_scale,
                 dq[i][4 * g + 3] * p.grad_scale);
  }
}

template <int D, int U, bool PAD>
static void launch(hipStream_t st, MaskedAttnParams const &p) {
  dim3 const grid((unsigned)(ceil_div(p.R, 128) * p.KH * p.B));
  bool const cap = p.capped != 0, bias = p.slopes != nullptr;
  if (cap && bias) masked_dq_heads_kernel<D, U, PAD, true, true><<<grid, 256, 0, st>>>(p);
  else if (cap) masked_dq_heads_kernel<D, U, PAD, true, false><<<grid, 256, 0, st>>>(p);
  else if (bias) masked_dq_heads_kernel<D, U, PAD, false, true><<<grid, 256, 0, st>>>(p);
  else masked_dq_heads_kernel<D, U, PAD, false, false><<<grid, 256, 0, st>>>(p);
}

hipError_t masked_attention_dq_heads(hipStream_t st, MaskedAttnParams const &p) {
  int const most = p.Dq > p.Dv ? p.Dq : p.Dv;
  if (p.Dq == p.Dv && p.Dq == 64) launch<64, 64, false>(st, p);
  else if (p.Dq == p.Dv && p.Dq == 128) launch<128, 128, false>(st, p);
  else if (most <= 64) launch<64, 64, true>(st, p);
  else if (most <= 96) launch<128, 96, true>(st, p);
  else launch<128, 128, true>(st, p);
  return hipGetLastError();
}

}  // namespace ffk
