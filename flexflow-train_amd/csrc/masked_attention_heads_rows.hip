// Masked attention, forward for few rows over bf16 heads up to 128 (see masked_attention.h for the mathematics and
// layouts).
//
// A workgroup is one wave: 32 rows of one key head (the query heads that share it among them) and a part of the keys.
// Bound by the bytes of K and V: the wave brings blocks of 32 keys into a ring of its own in LDS by direct loads, one
// block ahead, and waits for nothing but its own loads, no barrier anywhere; five such waves on a CU (heads of 128) keep
// 80 KB of requests in flight.  The parts of a row meet in masked_merge_kernel.  (One row of 32 heads on 8 key heads of
// 128, 16 sequences of 4096 to 8192 keys, 402 MB: four waves of one workgroup on tiles of 128 keys through registers, as
// in the general kernel, take 111 us, this kernel 86, and 81 by loads that keep nothing in the caches, 4.9 TB/s.)
#include "masked_attention_heads.h"

namespace ffk {

template <int D>
struct RowsFwd {
  static constexpr int kKeys = 32;
  static constexpr int kCPR = D / 8;               // 16-byte chunks of a row
  static constexpr int kRowsPerLoad = 64 / kCPR;
  static constexpr int kLoads = kKeys / kRowsPerLoad;  // direct loads, per tensor and block
  static constexpr int kBlock = kKeys * D;
  __device__ static int kswz(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
  __device__ static int vswz(int row) { return D == 128 ? (row & 3) : ((row >> 1) & 1); }
  static_assert(D == 64 || D == 128, "permutations are written for these two");
};

template <int D, int U, bool PAD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64) void masked_fwd_rows_kernel(MaskedAttnParams p) {
  using C = RowsFwd<D>;
  __shared__ __attribute__((aligned(1024))) bf16 Ks[2][C::kBlock];
  __shared__ __attribute__((aligned(1024))) bf16 Vs[2][C::kBlock];
  int const dim_qk = PAD ? p.Dq : D, dim_v = PAD ? p.Dv : D;  // the heads themselves
  int const lane = threadIdx.x, h32 = lane >> 5;
  int kh, b, hb;
  int const rest = place_of(p, kh, b, hb);
  int const split = rest % p.splits, rb = rest / p.splits;
  int const row = rb * 32 + (lane & 31);
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
  int const lo_all = wave_min_int(lo), hi_all = wave_max_int(hi);
  // rows that do not exist narrow nothing
  int const lo_max = wave_max_int(row < p.R ? lo : 0), hi_min = wave_min_int(row < p.R ? hi : 1 << 30);
  // this part of the window, in whole blocks: parts of one size for all rows of the launch, so that no workgroup has more
  // to read than another
  int const all_blocks = hi_all > lo_all ? (hi_all - lo_all + 31) / 32 : 0;
  int const per = ((p.Skv + 31) / 32 + p.splits - 1) / p.splits;
  int const first = min(split * per, all_blocks);
  int const nblocks = __builtin_amdgcn_readfirstlane(min(per, all_blocks - first));
  int const begin = __builtin_amdgcn_readfirstlane(lo_all + first * 32);
  bf16 const *kp = uniform_pointer(static_cast<bf16 const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * dim_qk);
  bf16 const *vp = uniform_pointer(static_cast<bf16 const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * dim_v);

  // Direct loads: lane l of load i writes LDS chunk 64 i + l and fetches the chunk that the permutation puts there.
  int const slot_row = lane / C::kCPR, slot_pc = lane % C::kCPR;
  int const v_lc = ((((slot_pc >> 2) ^ C::vswz(slot_row)) << 2) | (slot_pc & 3));
  static_assert(C::kRowsPerLoad % 4 == 0, "the permutation of V repeats from load to load");
  unsigned const ks_addr = lds_address_of(&Ks[0][0]), vs_addr = lds_address_of(&Vs[0][0]);
  unsigned k_voff[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; i++) {
    int const r = slot_row + i * C::kRowsPerLoad;
    k_voff[i] = tile_offset<PAD>(r * p.k_ss, (slot_pc ^ C::kswz(r)) * 8, dim_qk);
  }
  unsigned const v_voff = tile_offset<PAD>(slot_row * p.v_ss, v_lc * 8, dim_v);
  auto issue = [&](int kv0, int buf) {
    i32x4 const k_rsrc = tile_resource<PAD>(kp + (int64_t)kv0 * p.k_ss), v_rsrc = tile_resource<PAD>(vp + (int64_t)kv0 * p.v_ss);
    unsigned const k_dst = ks_addr + (unsigned)(buf * C::kBlock * 2), v_dst = vs_addr + (unsigned)(buf * C::kBlock * 2);
    if (kv0 + C::kKeys > hi_all) {  // uniform
      // keys past the last one that is seen repeat it: what lies there is not read
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        int const slot = slot_row + i * C::kRowsPerLoad, r = min(slot, hi_all - 1 - kv0);
        lds_dma16_once(k_rsrc, tile_offset<PAD>(r * p.k_ss, (slot_pc ^ C::kswz(slot)) * 8, dim_qk), 0u, k_dst + (unsigned)(i * 1024));
        lds_dma16_once(v_rsrc, tile_offset<PAD>(r * p.v_ss, v_lc * 8, dim_v), 0u, v_dst + (unsigned)(i * 1024));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        lds_dma16_once(k_rsrc, k_voff[i], 0u, k_dst + (unsigned)(i * 1024));
        lds_dma16_once(v_rsrc, v_voff, (unsigned)(i * C::kRowsPerLoad) * (unsigned)p.v_ss * 2u, v_dst + (unsigned)(i * 1024));
      }
    }
  };
  if (nblocks > 0) issue(begin, 0);

  bf16x8 qf[U / 16];
  {
    bf16 const *qp = static_cast<bf16 const *>(p.q) + (int64_t)b * p.q_bs + (int64_t)qi * p.q_ss + (int64_t)head * dim_qk;
#pragma unroll
    for (int kk = 0; kk < U / 16; kk++) qf[kk] = head_chunk<PAD>(qp, kk * 16 + h32 * 8, dim_qk);
  }
  f32x16 oacc[U / 32];
#pragma unroll
  for (int i = 0; i < U / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) oacc[i][r] = 0.0f;
  float m_run = -INFINITY, l_part = 0.0f;
  int k_off[U / 16], v_off[U / 32];
#pragma unroll
  for (int kk = 0; kk < U / 16; kk++) k_off[kk] = (lane & 31) * D + (((2 * kk + h32) ^ C::kswz(lane & 31)) << 3);
  {
    int const i16 = lane & 15, lr = 4 * h32 + (i16 >> 2);
#pragma unroll
    for (int i = 0; i < U / 32; i++) v_off[i] = lr * D + ((i ^ C::vswz(lr)) << 5) + ((lane >> 4) & 1) * 16 + (i16 & 3) * 4;
  }
  wait_all_vmem_known_to_compiler();  // the rows' operands: no wait for them inside the loop
  constexpr int kPerBlock = 2 * C::kLoads;
  auto block_step = [&](int n, auto buffer_tag) __attribute__((always_inline)) {
    constexpr int cur = decltype(buffer_tag)::value;
    int const kv0 = begin + n * 32;
    // past the end the last block is asked for again, into a buffer nobody reads: one wait count for all steps
    issue(begin + min(n + 1, nblocks - 1) * 32, cur ^ 1);
    wait_vmcnt<kPerBlock>();
    bf16 const *kt = Ks[cur], *vt = Vs[cur];
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < U / 16; kk++)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<bf16x8 const *>(kt + k_off[kk]), qf[kk], s, 0, 0, 0);
    int const kv_first = kv0 + 4 * h32;
    float const distance = (float)(position - kv_first);
#pragma unroll
    for (int r = 0; r < 16; r++) {
      s[r] = capped<CAP ? kCapLogistic : kNoCap>(p, s[r]);
      if constexpr (BIAS) s[r] = __builtin_fmaf(-slope, fabsf(distance - (float)(8 * (r >> 2) + (r & 3))), s[r]);
    }
    if (kv0 < lo_max || kv0 + 32 > hi_min) {  // uniform: not seen whole by all rows
      int const from = lo - kv_first, to = hi - kv_first;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        int const kv = 8 * (r >> 2) + (r & 3);
        s[r] = kv < from || kv >= to ? -INFINITY : s[r];
      }
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
    float const m_new = fmaxf(m_run, max_across_halves(mx) * p.score_scale);
    float const m_use = m_new == -INFINITY ? 0.0f : m_new;  // nothing seen yet: every exponential is 0
    // (a row that has seen nothing yet has only zeros to rescale)
    if (__builtin_amdgcn_ballot_w64(m_new != m_run && m_run != -INFINITY) != 0) {
      float const alpha = __builtin_amdgcn_exp2f(m_run - m_use);
      l_part *= alpha;
#pragma unroll
      for (int i = 0; i < U / 32; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[i][r] *= alpha;
    }
    m_run = m_new;
    float pv[16], sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      pv[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.score_scale, -m_use));
      sum += pv[r];
    }
    l_part += sum;
    bf16x8 const pf[2] = {pack8(pv), pack8(pv + 8)};
#pragma unroll
    for (int js = 0; js < 2; js++)
#pragma unroll
      for (int i = 0; i < U / 32; i++) {
        bf16 const *q = vt + v_off[i] + js * 16 * D;
        union {
          s16x4 h2[2];
          bf16x8 v;
        } u;
        u.h2[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(q));
        u.h2[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(q + 8 * D));
        oacc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.v, pf[js], oacc[i], 0, 0, 0);
      }
    // The reads of this buffer are over before the next step's loads write it: their results went into the MFMAs above,
    // which the wait below makes certain for the last of them.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  for (int n = 0; n < nblocks; n += 2) {
    block_step(n, std::integral_constant<int, 0>{});
    if (n + 1 < nblocks) block_step(n + 1, std::integral_constant<int, 1>{});
  }
  wait_vmcnt<0>();  // before the LDS is another workgroup's

  float const l = l_part + __shfl_xor(l_part, 32, 64);
  if (row >= p.R) return;
  if (p.splits > 1) {
    int64_t const at = ((int64_t)split * p.B * p.KH + hb) * p.R + row;
    float *po = p.part_o + at * dim_v;
#pragma unroll
    for (int i = 0; i < U / 32; i++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        if (!PAD || i * 32 + 8 * g + 4 * h32 < dim_v)
          store4(po + i * 32 + 8 * g + 4 * h32, oacc[i][4 * g], oacc[i][4 * g + 1], oacc[i][4 * g + 2], oacc[i][4 * g + 3]);
    if (h32 == 0) {
      p.part_ml[2 * at] = m_run;
      p.part_ml[2 * at + 1] = l;
    }
    return;
  }
  float const inv = l == 0.0f ? 0.0f : 1.0f / l;
  bf16 *op = static_cast<bf16 *>(p.o) + (int64_t)b * p.o_bs + (int64_t)qi * p.o_ss + (int64_t)head * dim_v;
#pragma unroll
  for (int i = 0; i < U / 32; i++)
#pragma unroll
    for (int g = 0; g < 4; g++)
      if (!PAD || i * 32 + 8 * g + 4 * h32 < dim_v)
        store4(op + i * 32 + 8 * g + 4 * h32, oacc[i][4 * g] * inv, oacc[i][4 * g + 1] * inv, oacc[i][4 * g + 2] * inv, oacc[i][4 * g + 3] * inv);
  if (h32 == 0 && p.lse != nullptr)
    p.lse[((int64_t)b * p.H + head) * p.Sq + qi] = l == 0.0f ? -INFINITY : (m_run + p.shift + __log2f(l)) * kLn2;
}

template <int D, int U, bool PAD>
static void launch(hipStream_t st, MaskedAttnParams const &p) {
  dim3 const grid((unsigned)(ceil_div(p.R, 32) * p.splits * p.KH * p.B));
  bool const cap = p.capped != 0, bias = p.slopes != nullptr;
  if (cap && bias) masked_fwd_rows_kernel<D, U, PAD, true, true><<<grid, 64, 0, st>>>(p);
  else if (cap) masked_fwd_rows_kernel<D, U, PAD, true, false><<<grid, 64, 0, st>>>(p);
  else if (bias) masked_fwd_rows_kernel<D, U, PAD, false, true><<<grid, 64, 0, st>>>(p);
  else masked_fwd_rows_kernel<D, U, PAD, false, false><<<grid, 64, 0, st>>>(p);
}

hipError_t masked_attention_fwd_rows(hipStream_t st, MaskedAttnParams const &p) {
  int const most = p.Dq > p.Dv ? p.Dq : p.Dv;
  if (p.Dq == p.Dv && p.Dq == 64) launch<64, 64, false>(st, p);
  else if (p.Dq == p.Dv && p.Dq == 128) launch<128, 128, false>(st, p);
  else if (most <= 64) launch<64, 64, true>(st, p);
  else if (most <= 96) launch<128, 96, true>(st, p);
  else launch<128, 128, true>(st, p);
  return hipGetLastError();
}

}  // namespace ffk
