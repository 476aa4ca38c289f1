// Masked attention, forward for bf16 heads up to 128 (see masked_attention.h for the mathematics and layouts).
//
// One workgroup takes 128 rows of one key head, 32 to a wave, and two workgroups run on a CU: the vector work of one
// wave (four instructions a score, ten with a cap and a bias) covers the matrix work of the other.  Keys and values
// come in tiles of 64 by direct loads, one tile ahead, and lie in LDS as in memory but for a permutation of the 16-byte
// chunks of a row on the fetching side, which keeps both ways of reading them free of bank conflicts.
//   The loop runs over the union of the rows' ranges.  A wave passes over a tile that none of its rows sees, and ranges
// are compared element by element only where a tile is not seen whole by all of its rows.
//   Bound by the issue of vector instructions: 8192 tokens, 16 heads of 128, causal, biased 330 us (0.83 PFLOP/s); 4 x 4096
// tokens in 3 documents, 32 heads of 128 on 8, causal, capped 367 us; 8 x 512 tokens in 4 documents, 16 heads of 64
// 18 us, where it is latency.  (For the second: vector steps fenced between the matrix instructions, as in the dK/dV
// kernel, 485 us; eight waves and three buffers 430.)
#include "masked_attention_heads.h"

namespace ffk {

template <int D>
struct HeadsFwd {
  static constexpr int kRows = 128, kKeys = 64;
  static constexpr int kCPR = D / 8;
  static constexpr int kLoads = kKeys * kCPR / 256;
  static constexpr int kRowsPerLoad = 256 / kCPR;
  static constexpr int kTile = kKeys * D;
  __device__ static int kswz(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
  __device__ static int vswz(int row) { return D == 128 ? (row & 3) : ((row >> 1) & 1); }
  static_assert(D == 64 || D == 128, "permutations are written for these two");
};

template <int D, int U, bool PAD, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 2) void masked_fwd_heads_kernel(MaskedAttnParams p) {
  using C = HeadsFwd<D>;
  __shared__ __attribute__((aligned(1024))) bf16 Ks[2][C::kTile];
  __shared__ __attribute__((aligned(1024))) bf16 Vs[2][C::kTile];
  __shared__ int window[2][4];
  int const dim_qk = PAD ? p.Dq : D, dim_v = PAD ? p.Dv : D;  // the heads themselves
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int const nrb = (p.R + C::kRows - 1) / C::kRows;
  int kh, b, hb;
  int const rb = nrb - 1 - place_of(p, kh, b, hb);  // under a causal mask the heaviest rows go first
  int const row = rb * C::kRows + wave * 32 + (lane & 31);
  int qi, qg;
  row_of(p, min(row, p.R - 1), qi, qg);
  int const head = kh * p.G + qg, position = p.q_offset + qi;
  int lo, hi;
  row_range(p, b, qi, lo, hi);
  if (row >= p.R) {
    lo = 1 << 30;
    hi = 0;
  }
  float slope = 0.0f;
  if constexpr (BIAS) slope = p.slopes[head] * p.slope_unit;
  int const w_lo_min = wave_min_int(lo), w_hi_max = wave_max_int(hi);
  // rows that do not exist narrow nothing
  int const w_lo_max = wave_max_int(row < p.R ? lo : 0), w_hi_min = wave_min_int(row < p.R ? hi : 1 << 30);
  if (lane == 0) {
    window[0][wave] = w_lo_min;
    window[1][wave] = w_hi_max;
  }
  __syncthreads();
  int const lo_all = __builtin_amdgcn_readfirstlane(min(min(window[0][0], window[0][1]), min(window[0][2], window[0][3])));
  int const hi_all = __builtin_amdgcn_readfirstlane(max(max(window[1][0], window[1][1]), max(window[1][2], window[1][3])));
  int const ntiles = hi_all > lo_all ? (hi_all - lo_all + C::kKeys - 1) / C::kKeys : 0;
  bf16 const *kp = uniform_pointer(static_cast<bf16 const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * dim_qk);
  bf16 const *vp = uniform_pointer(static_cast<bf16 const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * dim_v);

  // Q as the B operand of S^T = K Q^T: column = row, k = d
  bf16x8 qf[U / 16];
  {
    bf16 const *qp = static_cast<bf16 const *>(p.q) + (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * dim_qk;
#pragma unroll
    for (int kk = 0; kk < U / 16; kk++) qf[kk] = head_chunk<PAD>(qp, kk * 16 + h32 * 8, dim_qk);
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
    k_voff[i] = tile_offset<PAD>((slot_row + i * C::kRowsPerLoad) * p.k_ss, k_lc * 8, dim_qk);
    v_voff[i] = tile_offset<PAD>((slot_row + i * C::kRowsPerLoad) * p.v_ss, v_lc * 8, dim_v);
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
        lds_dma16(k_rsrc, tile_offset<PAD>(r * p.k_ss, k_lc * 8, dim_qk), 0u, k_dst + (unsigned)(i * 4096));
      }
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        int const r = min(slot_row + i * C::kRowsPerLoad, hi_all - 1 - kv0);
        lds_dma16(v_rsrc, tile_offset<PAD>(r * p.v_ss, v_lc * 8, dim_v), 0u, v_dst + (unsigned)(i * 4096));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) lds_dma16(k_rsrc, k_voff[i], 0u, k_dst + (unsigned)(i * 4096));
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) lds_dma16(v_rsrc, v_voff[i], 0u, v_dst + (unsigned)(i * 4096));
    }
  };

  f32x16 oacc[U / 32];
#pragma unroll
  for (int i = 0; i < U / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) oacc[i][r] = 0.0f;
  float m_run = -INFINITY;
  float l_part = 0.0f;  // this lane's 16 of every 32 keys; the two lane halves meet at the end

  // K fragment (key block j, d step kk): row j*32 + l%32, chunk (2 kk + l/32) ^ kswz(row)
  int k_off[U / 16];
#pragma unroll
  for (int kk = 0; kk < U / 16; kk++) k_off[kk] = (lane & 31) * D + (((2 * kk + h32) ^ C::kswz(lane & 31)) << 3);
  // V fragment (d block i): rows 4 (l/32) + (l%16)/4 (+ 8) of a 16-row step, 4 columns at 16 ((l/16)%2) + 4 (l%4)
  int v_off[U / 32];
  {
    int const i16 = lane & 15, lr = 4 * h32 + (i16 >> 2);
#pragma unroll
    for (int i = 0; i < U / 32; i++) v_off[i] = lr * D + ((i ^ C::vswz(lr)) << 5) + ((lane >> 4) & 1) * 16 + (i16 & 3) * 4;
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
  // With a bias from the last tile to the first: under a causal mask the largest scores come first then, and the reference
  // point stays where it is (the other way round it moves in every tile: 8192 tokens, 16 heads of 128, 395 us and 330).
  // Without one from the first: the workgroups of a head read the same keys at about the same time (4 sequences of 4096 in
  // 3 documents each, 32 heads on 8 of 128, a cap: 374 us, the other way round 396).
  auto tile_at = [&](int it) { return lo_all + (BIAS ? ntiles - 1 - it : it) * C::kKeys; };
  if (ntiles > 0) issue_tile(tile_at(0), 0);
  wait_all_vmem_known_to_compiler();  // the Q fragments too: no wait for them inside the loop
  __syncthreads();
  // One tile that this wave works on; edge (uniform): one that is not seen whole by all of its rows.
  auto tile_work = [&](int kv0, bf16 const *kt, bf16 const *vt, bool edge) __attribute__((always_inline)) {
    f32x16 s[2];
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) s[j][r] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < U / 16; kk++)
#pragma unroll
      for (int j = 0; j < 2; j++) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(kt, j, kk), qf[kk], s[j], 0, 0, 0);
    int const kv_first = kv0 + 4 * h32;
    if constexpr (CAP || BIAS) {
      float const distance = (float)(position - kv_first);
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[j][r] = capped<CAP ? kCapLogistic : kNoCap>(p, s[j][r]);
          if constexpr (BIAS) s[j][r] = __builtin_fmaf(-slope, fabsf(distance - (float)(j * 32 + 8 * (r >> 2) + (r & 3))), s[j][r]);
        }
    }
    if (edge) {
      int const from = lo - kv_first, to = hi - kv_first;
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          int const kv = j * 32 + 8 * (r >> 2) + (r & 3);
          s[j][r] = kv < from || kv >= to ? -INFINITY : s[j][r];
        }
    }
    float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; r++) mx = fmaxf(fmaxf(mx, s[0][r]), s[1][r]);
    // (score_scale is positive, so it commutes with the maximum.)  The reference point of the exponentials moves only
    // when the maximum has grown by more than kLazy (in powers of two): until then probabilities may exceed 1, by at most
    // 2^kLazy, harmless in 32-bit sums and in bf16's range, and nearly no tile rescales the accumulators.
    constexpr float kLazy = 8.0f;
    float const m = max_across_halves(mx) * p.score_scale;
    float const m_new = m > m_run + kLazy ? m : m_run;
    float const m_use = m_new == -INFINITY ? 0.0f : m_new;  // nothing seen yet: every exponential is 0
    // (a row that has seen nothing yet has only zeros to rescale)
    if (__builtin_amdgcn_ballot_w64(m_new != m_run && m_run != -INFINITY) != 0) {
      float const alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_use);
      l_part *= alpha;
      mma_settled(oacc);
#pragma unroll
      for (int i = 0; i < U / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[i][r] *= alpha;
#pragma unroll
      for (int i = 0; i < U / 32; i++) asm volatile("" : "+a"(oacc[i]));
    }
    m_run = m_new;
    bf16x8 pf[4];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float pv[16];
#pragma unroll
      for (int r = 0; r < 16; r++) {
        pv[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], p.score_scale, -m_use));
        sum += pv[r];
      }
      pf[2 * j] = pack8(pv);
      pf[2 * j + 1] = pack8(pv + 8);
    }
    l_part += sum;
    bf16x8 vf[4];  // a fragment is read three MFMAs ahead of its use
#pragma unroll
    for (int n = 0; n < 3; n++) vf[n] = v_frag(vt, n / (U / 32), n % (U / 32));
    asm volatile("s_nop 3" : "+v"(pf[0]), "+v"(pf[1]), "+v"(pf[2]), "+v"(pf[3]));
#pragma unroll
    for (int n = 0; n < U / 8; n++) {
      if (n + 3 < U / 8) vf[(n + 3) % 4] = v_frag(vt, (n + 3) / (U / 32), (n + 3) % (U / 32));
      mma_kept(oacc[n % (U / 32)], vf[n % 4], pf[n / (U / 32)]);
    }
  };
  auto tile_step = [&](int it, auto buffer_tag) __attribute__((always_inline)) {
    constexpr int cur = decltype(buffer_tag)::value;
    int const kv0 = tile_at(it);
    if (it + 1 < ntiles) issue_tile(tile_at(it + 1), cur ^ 1);
    if (kv0 < w_hi_max && kv0 + C::kKeys > w_lo_min) {
      tile_work(kv0, Ks[cur], Vs[cur], kv0 < w_lo_max || kv0 + C::kKeys > w_hi_min);
    }
    wait_vmcnt<0>();  // this wave's part of the next tile has landed
    __syncthreads();
  };
  for (int it = 0; it < ntiles; it += 2) {
    tile_step(it, std::integral_constant<int, 0>{});
    if (it + 1 < ntiles) tile_step(it + 1, std::integral_constant<int, 1>{});
  }

  mma_settled(oacc);
  float const l = l_part + __shfl_xor(l_part, 32, 64);
  if (row < p.R) {
    float const inv = l == 0.0f ? 0.0f : 1.0f / l;
    bf16 *op = static_cast<bf16 *>(p.o) + (int64_t)b * p.o_bs + (int64_t)qi * p.o_ss + (int64_t)head * dim_v;
#pragma unroll
    for (int i = 0; i < U / 32; i++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        if (!PAD || i * 32 + 8 * g + 4 * h32 < dim_v)
          store4(op + i * 32 + 8 * g + 4 * h32, oacc[i][4 * g] * inv, oacc[i][4 * g + 1] * inv, oacc[i][4 * g + 2] * inv,
                 oacc[i][4 * g + 3] * inv);
    if (h32 == 0 && p.lse != nullptr)
      p.lse[((int64_t)b * p.H + head) * p.Sq + qi] = l == 0.0f ? -INFINITY : (m_run + p.shift + __log2f(l)) * kLn2;
  }
}

template <int D, int U, bool PAD>
static void launch(hipStream_t st, MaskedAttnParams const &p) {
  dim3 const grid((unsigned)(ceil_div(p.R, HeadsFwd<D>::kRows) * p.KH * p.B));
  bool const cap = p.capped != 0, bias = p.slopes != nullptr;
  if (cap && bias) masked_fwd_heads_kernel<D, U, PAD, true, true><<<grid, 256, 0, st>>>(p);
  else if (cap) masked_fwd_heads_kernel<D, U, PAD, true, false><<<grid, 256, 0, st>>>(p);
  else if (bias) masked_fwd_heads_kernel<D, U, PAD, false, true><<<grid, 256, 0, st>>>(p);
  else masked_fwd_heads_kernel<D, U, PAD, false, false><<<grid, 256, 0, st>>>(p);
}

hipError_t masked_attention_fwd_heads(hipStream_t st, MaskedAttnParams const &p) {
  int const most = p.Dq > p.Dv ? p.Dq : p.Dv;
  if (p.Dq == p.Dv && p.Dq == 64) launch<64, 64, false>(st, p);
  else if (p.Dq == p.Dv && p.Dq == 128) launch<128, 128, false>(st, p);
  else if (most <= 64) launch<64, 64, true>(st, p);
  else if (most <= 96) launch<128, 96, true>(st, p);
  else launch<128, 128, true>(st, p);
  return hipGetLastError();
}

}  // namespace ffk
