// Masked attention, dK and dV for bf16 heads up to 128 (see masked_attention.h for the mathematics and layouts).
//
// One workgroup owns 128 keys of one key head, 32 to a wave, whose K and V rows are MFMA operands in registers for the
// whole kernel next to the accumulators; one wave runs on a SIMD.  It streams the rows of all query heads that read the key
// head in tiles of 64, two halves of 32: Q, dO and what the dQ kernel left of the rows arrive by direct loads in three LDS
// buffers, two tiles ahead.  Vector and matrix work overlap inside the wave: behind every MFMA sits one step each of a few
// scores (fenced against the scheduler), and every LDS fragment is read a few MFMAs ahead of its use, through the ends of
// the phases too.  A vector instruction that needs the one right in front of it waits: a lone wave issues one in 10 cycles
// then, and one in 6 otherwise, which is why a score takes its steps in different slots.  The accumulators stay in accumulation registers (mma_kept);
// everything else, 200 registers of operands, scores and fragments, has the ordinary ones.
//   Which tiles: a list in LDS of those with a row that sees one of the 128 keys, from the summaries of ranges, made for
// 512 tiles at a time.  A wave passes over a tile none of whose rows sees its 32 keys, and compares ranges element by
// element only where not all rows see all of them.  Rows that see none of the 128 keys are cleared in LDS before use: what
// lies in them must not meet the zeros of the masked probabilities; so is the Q of those that see one key.
//   A tile lies in LDS as in memory, [64 rows][D], the 16-byte chunks of a row permuted on the fetching side such that
// both ways it is read (16 bytes a lane by rows, and turned) are free of bank conflicts.
//   8192 tokens, 16 heads of 128, causal, biased 630 us (0.87 PFLOP/s with its four products); 4 x 4096 tokens in 3 documents,
// 32 heads of 128 on 8, causal, capped 680 us; 8 x 512 tokens in 4 documents, 16 heads of 64 23 us.
#include "masked_attention_heads.h"

namespace ffk {

template <int D>
struct HeadsDkdv {
  static constexpr int kKeys = 128, kRows = 64;
  static constexpr int kCPR = D / 8;                // 16-byte chunks of a row
  static constexpr int kLoads = kRows * kCPR / 256; // direct loads of a thread, per tensor and tile
  static constexpr int kRowsPerLoad = 256 / kCPR;
  static constexpr int kTile = kRows * D;
  static constexpr int kList = 512;  // tiles listed at a time
  static_assert(D == 64 || D == 128, "permutations are written for these two");
  __device__ static int swz(int row) {
    return D == 128 ? (((row & 3) << 2) | ((row >> 2) & 3)) : ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
  }
};

template <int D, bool PAD, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) void masked_dkdv_heads_kernel(MaskedAttnParams p) {
  using C = HeadsDkdv<D>;
  constexpr int NBUF = 3;
  __shared__ __attribute__((aligned(1024))) bf16 Qs[NBUF][C::kTile];
  __shared__ __attribute__((aligned(1024))) bf16 Gs[NBUF][C::kTile];
  __shared__ __attribute__((aligned(256))) float Rows[NBUF][BIAS ? 6 : 4][64];  // the fields of a tile's rows
  __shared__ __attribute__((aligned(256))) float Unused[64];
  __shared__ int list_tile[C::kList];
  __shared__ RangeSummary list_sum[C::kList];
  __shared__ int wave_count[4];
  int const dim_qk = PAD ? p.Dq : D, dim_v = PAD ? p.Dv : D;  // the heads themselves
  int const t = threadIdx.x, lane = t & 63, h32 = lane >> 5;
  int const wave = __builtin_amdgcn_readfirstlane(t >> 6);
  int kh, b, hb;
  int const kv0 = place_of(p, kh, b, hb) * C::kKeys;  // under a causal mask the first keys are seen by most rows
  int const wkv0 = kv0 + wave * 32, kvcol = wkv0 + (lane & 31);
  bf16 const *qp = static_cast<bf16 const *>(p.q) + (int64_t)b * p.q_bs + (int64_t)kh * p.G * dim_qk;
  bf16 const *gp = static_cast<bf16 const *>(p.d_o) + (int64_t)b * p.o_bs + (int64_t)kh * p.G * dim_v;
  bf16 const *kp = static_cast<bf16 const *>(p.k) + (int64_t)b * p.k_bs + (int64_t)kh * dim_qk;
  bf16 const *vp = static_cast<bf16 const *>(p.v) + (int64_t)b * p.v_bs + (int64_t)kh * dim_v;
  float const *rowp = p.rows + (int64_t)hb * kRowFields * p.padded_rows;

  bf16x8 kf[D / 16], vf[D / 16];
  {
    int const r = min(kvcol, p.Skv - 1);
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++) {
      kf[kk] = head_chunk<PAD>(kp + (int64_t)r * p.k_ss, kk * 16 + h32 * 8, dim_qk);
      vf[kk] = head_chunk<PAD>(vp + (int64_t)r * p.v_ss, kk * 16 + h32 * 8, dim_v);
    }
  }
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      dk[i][r] = 0.0f;
      dv[i][r] = 0.0f;
    }

  // Direct loads of a tile: thread slot c (of 256 a load) writes LDS chunk c of the load's 4 KB and fetches the chunk that
  // the permutation puts there.  The rows' fields: one load of 64 values to each wave (two with slopes and positions;
  // waves 2 and 3 then fetch theirs a second time to where nobody reads), so that one wait count fits all waves.
  int const slot_row = t / C::kCPR, slot_lc = (t % C::kCPR) ^ C::swz(t / C::kCPR);
  unsigned const qs_addr = lds_address_of(&Qs[0][0]), gs_addr = lds_address_of(&Gs[0][0]), rows_addr = lds_address_of(&Rows[0][0][0]);
  unsigned const unused_addr = lds_address_of(&Unused[0]);
  i32x4 const rq = tile_resource<PAD>(qp), rg = tile_resource<PAD>(gp);
  i32x4 const rr = buffer_resource(rowp + (int64_t)wave * p.padded_rows);
  i32x4 const rx = buffer_resource(rowp + (int64_t)(kRowSlope + (wave & 1)) * p.padded_rows);
  constexpr int kFields = BIAS ? 6 : 4;
  constexpr int kLoadsPerTile = 2 * C::kLoads + (BIAS ? 2 : 1);
  // Where G divides 64, a tile's rows lie as its first row's does, and the lanes' offsets inside it never change.
  bool const even = p.group.d <= 64 && 64 % p.group.d == 0;
  unsigned q_off[C::kLoads], g_off[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; i++) {
    int qi, g;
    row_of(p, slot_row + i * C::kRowsPerLoad, qi, g);
    q_off[i] = row_offset<PAD>((unsigned)qi * ((unsigned)p.q_ss * 2u), g, slot_lc * 8, dim_qk);
    g_off[i] = row_offset<PAD>((unsigned)qi * ((unsigned)p.o_ss * 2u), g, slot_lc * 8, dim_v);
  }
  auto issue_tile = [&](int row0, int buf) {
    unsigned const dst = (unsigned)(buf * C::kTile * 2 + wave * 1024);
    if (even && row0 + C::kRows <= p.R) {  // uniform
      unsigned const first = __builtin_amdgcn_readfirstlane(p.group.div((uint32_t)row0));
      unsigned const q_tile = first * ((unsigned)p.q_ss * 2u), g_tile = first * ((unsigned)p.o_ss * 2u);
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        lds_dma16(rq, q_off[i], q_tile, qs_addr + dst + (unsigned)(i * 4096));
        lds_dma16(rg, g_off[i], g_tile, gs_addr + dst + (unsigned)(i * 4096));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::kLoads; i++) {
        int qi, g;
        row_of(p, min(row0 + slot_row + i * C::kRowsPerLoad, p.R - 1), qi, g);
        lds_dma16(rq, row_offset<PAD>((unsigned)qi * ((unsigned)p.q_ss * 2u), g, slot_lc * 8, dim_qk), 0u, qs_addr + dst + (unsigned)(i * 4096));
        lds_dma16(rg, row_offset<PAD>((unsigned)qi * ((unsigned)p.o_ss * 2u), g, slot_lc * 8, dim_v), 0u, gs_addr + dst + (unsigned)(i * 4096));
      }
    }
    unsigned const at = (unsigned)(row0 + lane) * 4u;  // padded_rows is whole tiles
    lds_dma4(rr, at, 0u, rows_addr + (unsigned)(buf * kFields + wave) * 256u);
    if constexpr (BIAS)
      lds_dma4(rx, at, 0u, wave >= 2 ? unused_addr : rows_addr + (unsigned)(buf * kFields + kRowSlope + wave) * 256u);
  };

  // Per-lane LDS offsets (in elements) of the two ways a tile is read (32 rows from its first row on).
  int row_off[D / 16], tr_off[D / 32][2];
  {
    int const r = lane & 31;
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++) row_off[kk] = r * D + (((2 * kk + h32) ^ C::swz(r)) << 3);
    int const i16 = lane & 15, q = i16 >> 2, bb = (lane >> 4) & 1, c = i16 & 3;
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
      for (int sec = 0; sec < 2; sec++) {
        int const row = 8 * sec + 4 * h32 + q, chunk = 4 * i + 2 * bb + (c >> 1);
        tr_off[i][sec] = row * D + ((chunk ^ C::swz(row)) << 3) + 4 * (c & 1);
      }
  }
  auto turned = [&](bf16 const *tile, int s, int i) __attribute__((always_inline)) -> bf16x8 {
    union {
      s16x4 h2[2];
      bf16x8 v;
    } u;
    u.h2[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tile + tr_off[i][0] + 16 * s * D));
    u.h2[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tile + tr_off[i][1] + 16 * s * D));
    return u.v;
  };

  // One tile that this wave works on; edge (uniform): one whose rows do not all see all of the wave's keys.
  auto tile_work = [&](bf16 const *qt, bf16 const *gt, float const *fields, bool edge) __attribute__((always_inline)) {
    constexpr int NM = D / 8;     // MFMAs of a phase
    constexpr int UPM = 16 / NM;  // units of vector work behind each
    constexpr int kAhead = 4;     // an LDS fragment is read this many MFMAs ahead of its use
    constexpr int NI = D / 32;
    // Fragment n of the tile's 4 NM.  Phases 0 and 1: S = Q K^T, then dP = dO V^T, of half 0, then 1 (rows = its 32 rows,
    // column = key): d step m of Q, or m - NM / 2 of dO.  Phases 2 and 3: dV += P^T dO and dK += dS^T Q of half 0, then 1:
    // step m / (2 NI), d block (m / 2) % NI of dO (m even) or of Q.
    auto fragment = [&](auto nc) __attribute__((always_inline)) -> bf16x8 {
      constexpr int n = decltype(nc)::value;
      constexpr int phase = n / NM, m = n % NM, h = phase & 1;
      if constexpr (phase < 2) return *reinterpret_cast<bf16x8 const *>((m >= NM / 2 ? gt : qt) + h * 32 * D + row_off[m % (NM / 2)]);
      else return turned(((m & 1) ? qt : gt) + h * 32 * D, m / (2 * NI), (m >> 1) % NI);
    };
    f32x16 s[2], dp[2];
    union {
      uint32_t u[4];
      bf16x8 v;
    } pa[2][2], da[2][2];  // P and dS of a half as operands: step s2 takes scores 8 s2 .. + 7
    // A score's steps, each of a vector instruction or two that do not need each other; s becomes P and dp becomes dS.
    f32x4 lrow[2][4], drow[2][4], srow[2][4];
    i32x4 prow[2][4];
    float far[2][16], y[2][16];
    constexpr int kBias = BIAS ? 1 : 0;
    constexpr int kScore = CAP ? 4 : BIAS ? 2 : 0;  // the step in which a score's y is there
    constexpr int kPack = D == 64 ? 0 : 1;  // a slot of its own (at two scores a slot there is none left)
    constexpr int kSteps = kScore + kBias + 3 + kPack;
    auto step = [&](auto hc, auto uc, auto kc) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value, u = decltype(uc)::value, k = decltype(kc)::value, g = u >> 2, e = u & 3;
      // the distance beside the first steps
      if constexpr (BIAS && k == 0) far[h][u] = __builtin_bit_cast(float, prow[h][g][e] - kvcol);
      if constexpr (BIAS && k == 1) far[h][u] = (float)__builtin_bit_cast(int, far[h][u]);
      if constexpr (CAP && k == 0) s[h][u] *= p.cap_in;
      if constexpr (CAP && k == 1) s[h][u] = __builtin_amdgcn_exp2f(s[h][u]);
      if constexpr (CAP && k == 2) s[h][u] += 1.0f;
      if constexpr (CAP && k == 3) s[h][u] = __builtin_amdgcn_rcpf(s[h][u]);  // capped<kCapLogistic>
      if constexpr (k == kScore && CAP) y[h][u] = __builtin_fmaf(-s[h][u], s[h][u], s[h][u]);  // capped_slope<kCapLogistic>
      if constexpr (k == kScore && BIAS) s[h][u] = __builtin_fmaf(-srow[h][g][e], fabsf(far[h][u]), s[h][u]);
      if constexpr (k == kScore + kBias) s[h][u] = __builtin_fmaf(s[h][u], p.score_scale, -lrow[h][g][e]);
      if constexpr (k == kScore + kBias) dp[h][u] -= drow[h][g][e];
      if constexpr (k == kScore + kBias + 1) s[h][u] = __builtin_amdgcn_exp2f(s[h][u]);
      if constexpr (k == kScore + kBias + 1 && CAP) dp[h][u] *= y[h][u];
      if constexpr (k == kScore + kBias + 2) dp[h][u] *= s[h][u];
      if constexpr (k == kSteps - 1 && (u & 1) == 1) {
        pa[h][u >> 3].u[(u & 7) >> 1] = pack_bf16x2(s[h][u - 1], s[h][u]);
        da[h][u >> 3].u[(u & 7) >> 1] = pack_bf16x2(dp[h][u - 1], dp[h][u]);
      }
    };
    // What rows 8 g + 4 (l/32) .. + 3 of a half bring along, four scores' worth.
    auto read_fields = [&](auto hc, auto gc) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value, g = decltype(gc)::value;
      int const at = h * 32 + 8 * g + 4 * h32;
      lrow[h][g] = *reinterpret_cast<f32x4 const *>(fields + kRowLse2 * 64 + at);
      drow[h][g] = *reinterpret_cast<f32x4 const *>(fields + kRowDelta * 64 + at);
      if constexpr (BIAS) {
        srow[h][g] = *reinterpret_cast<f32x4 const *>(fields + kRowSlope * 64 + at);
        prow[h][g] = *reinterpret_cast<i32x4 const *>(fields + kRowPosition * 64 + at);
      }
    };
    // What a row does not see becomes 0 in the finished operands, by their bits: whatever it was.  (A second instance of the
    // whole tile for the masked ones makes the compiler move the accumulators where the two meet.)
    auto mask = [&](auto hc, auto sc) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value, s2 = decltype(sc)::value;
      int const *row_lo = reinterpret_cast<int const *>(fields + kRowLo * 64), *row_hi = reinterpret_cast<int const *>(fields + kRowHi * 64);
#pragma unroll
      for (int g = 2 * s2; g < 2 * s2 + 2; g++) {
        i32x4 const lo4 = *reinterpret_cast<i32x4 const *>(row_lo + h * 32 + 8 * g + 4 * h32);
        i32x4 const hi4 = *reinterpret_cast<i32x4 const *>(row_hi + h * 32 + 8 * g + 4 * h32);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          uint32_t const keep = (kvcol < lo4[e] || kvcol >= hi4[e] ? 0u : 0xffffu) | (kvcol < lo4[e + 1] || kvcol >= hi4[e + 1] ? 0u : 0xffff0000u);
          pa[h][s2].u[2 * (g & 1) + e / 2] &= keep;
          da[h][s2].u[2 * (g & 1) + e / 2] &= keep;
        }
      }
      // the wait states between a vector instruction and mma_kept
      asm volatile("s_nop 3" : "+v"(pa[h][s2].v), "+v"(da[h][s2].v));
    };
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        s[h][r] = 0.0f;
        dp[h][r] = 0.0f;
      }
    bf16x8 fr[kAhead + 1];
    static_for<0, kAhead>([&](auto nc) { fr[decltype(nc)::value] = fragment(nc); });
    static_for<0, 4 * NM>([&](auto nc) {
      constexpr int n = decltype(nc)::value;
      constexpr int phase = n / NM, m = n % NM, h = phase & 1;
      // The scores of half h are in steps from slot kFirst + NM h on, UPM of them entering a slot: S is there since slot
      // NM / 2 - 1 + NM h, and dP, which a score needs kScore + kBias steps on, since slot NM - 1 + NM h.  P and dS of a
      // half's step s2 are needed from slot (2 + h) NM + s2 NM / 2 on.
      constexpr int kNeedsDp = NM + 1 - kScore - kBias, kNeedsS = NM / 2 + NM / 8;
      constexpr int kFirst = kNeedsDp > kNeedsS ? kNeedsDp : kNeedsS;
      static_assert(kFirst + 15 / UPM + kSteps <= 2 * NM + NM / 2 && kFirst + 7 / UPM + kSteps <= 2 * NM, "operands are ready");
      if constexpr (phase >= 2 && m % (NM / 2) == 0) {
        if (edge) mask(std::integral_constant<int, h>{}, std::integral_constant<int, m / (NM / 2)>{});
      }
      bf16x8 const f = fr[n % (kAhead + 1)];
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (phase < 2) {
        if constexpr (m < NM / 2) s[h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, kf[m], s[h], 0, 0, 0);
        else dp[h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, vf[m - NM / 2], dp[h], 0, 0, 0);
      } else {
        constexpr int s2 = m / (2 * NI), i = (m / 2) % NI;
        if constexpr (m % 2 == 0) mma_kept(dv[i], pa[h][s2].v, f);
        else mma_kept(dk[i], da[h][s2].v, f);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n + kAhead < 4 * NM) fr[(n + kAhead) % (kAhead + 1)] = fragment(std::integral_constant<int, n + kAhead>{});
      static_for<0, 2>([&](auto hc) {
        // this slot's place in the half's sequence, and the fields of the scores that enter three slots on
        constexpr int at = n - kFirst - NM * decltype(hc)::value;
        if constexpr (at + 3 >= 0 && (at + 3) * UPM < 16 && (at + 3) * UPM % 4 == 0)
          read_fields(hc, std::integral_constant<int, (at + 3) * UPM / 4>{});
        // the last steps of the oldest scores first
        static_for<0, kSteps>([&](auto rc) {
          constexpr int k = kSteps - 1 - decltype(rc)::value;
          if constexpr (at - k >= 0 && (at - k) * UPM < 16)
            static_for<0, UPM>([&](auto vc) { step(hc, std::integral_constant<int, (at - k) * UPM + decltype(vc)::value>{}, std::integral_constant<int, k>{}); });
        });
      });
    });
    __builtin_amdgcn_sched_barrier(0);
  };

  int const nsum = (p.R + 31) / 32, ntiles = (p.R + 63) / 64;
  RangeSummary const *sums = p.summary + (int64_t)b * nsum;
  for (int chunk = 0; chunk < ntiles; chunk += C::kList) {
    // the tiles of this chunk that are worked on, in order
    int count = 0;
#pragma unroll
    for (int part = 0; part < C::kList / 256; part++) {
      int const tile = chunk + part * 256 + t;
      RangeSummary s = {1 << 30, 0, 1 << 30, 0};
      if (tile < ntiles) {
        s = sums[2 * tile];
        RangeSummary const s1 = 2 * tile + 1 < nsum ? sums[2 * tile + 1] : RangeSummary{1 << 30, 0, 1 << 30, 0};
        s = RangeSummary{min(s.lo_min, s1.lo_min), max(s.hi_max, s1.hi_max), max(s.lo_max, s1.lo_max), min(s.hi_min, s1.hi_min)};
      }
      bool const wanted = s.lo_min < kv0 + C::kKeys && s.hi_max > kv0;
      uint64_t const mask = __builtin_amdgcn_ballot_w64(wanted);
      __syncthreads();  // the counts (and, in the first part, the lists) are free
      if (lane == 0) wave_count[wave] = __builtin_popcountll(mask);
      __syncthreads();
      int at = count;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        int const n = __builtin_amdgcn_readfirstlane(wave_count[w]);
        if (w < wave) at += n;
        count += n;
      }
      if (wanted) {
        at += __builtin_popcountll(mask & ((1ull << lane) - 1));
        list_tile[at] = tile;
        list_sum[at] = s;
      }
    }
    __syncthreads();
    if (count == 0) continue;  // uniform

    auto row0_of = [&](int n) { return __builtin_amdgcn_readfirstlane(list_tile[n]) * C::kRows; };
    issue_tile(row0_of(0), 0);
    issue_tile(row0_of(min(1, count - 1)), 1);
    int next_row0 = row0_of(min(2, count - 1));
    int next_tile = list_tile[min(3, count - 1)];
    RangeSummary sum = list_sum[0];
    // tiles 0 and 1 have landed, and so have the K and V fragments: told to the compiler
    wait_all_vmem_known_to_compiler();
    __syncthreads();
    int cur = 0;
    for (int it = 0; it < count; it++) {
      // buffer (it+2) % 3 was read during step it-1; every wave has passed the barrier that ended it.  Past the end the last
      // tile is fetched again into a buffer nobody reads: the count of loads in flight is the same at every wait.
      issue_tile(next_row0, cur == 0 ? 2 : cur - 1);
      int const lo_min = __builtin_amdgcn_readfirstlane(sum.lo_min), hi_max = __builtin_amdgcn_readfirstlane(sum.hi_max);
      int const lo_max = __builtin_amdgcn_readfirstlane(sum.lo_max), hi_min = __builtin_amdgcn_readfirstlane(sum.hi_min);
      // the list's entries of the tiles to come, read a step ahead of their use
      next_row0 = __builtin_amdgcn_readfirstlane(next_tile) * C::kRows;
      next_tile = list_tile[min(it + 4, count - 1)];
      sum = list_sum[min(it + 1, count - 1)];
      bf16 *qt = Qs[cur], *gt = Gs[cur];
      float const *fields = &Rows[cur][0][0];
      if (lo_max >= kv0 + C::kKeys || hi_min <= kv0) {  // uniform: a row here sees none of the keys, or one alone
        int at = t;
        // Nothing of the addresses below is held in registers through the loop: with it heads of 64 pass the 256 that leave a
        // SIMD two waves (a pass over 8 x 512 tokens in 4 documents 73 us, and 64).
        asm volatile("" : "+v"(at));
        int const row = at >> 2, row_lo = __float_as_int(fields[kRowLo * 64 + row]), row_hi = __float_as_int(fields[kRowHi * 64 + row]);
        bool const none = row_lo >= kv0 + C::kKeys || row_hi <= kv0;
        if (none || one_key(row_lo, row_hi)) {
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            int const chunk = row * D + (c * 4 + (at & 3)) * 8;
            *reinterpret_cast<u32x4 *>(qt + chunk) = u32x4{0u, 0u, 0u, 0u};
            if (none) *reinterpret_cast<u32x4 *>(gt + chunk) = u32x4{0u, 0u, 0u, 0u};
          }
        }
        __syncthreads();
      }
      if (lo_min < wkv0 + 32 && hi_max > wkv0) {
        tile_work(qt, gt, fields, lo_max > wkv0 || hi_min < wkv0 + 32);
      }
      wait_vmcnt<kLoadsPerTile>();  // this wave's part of the next tile has landed
      __syncthreads();
      cur = cur == 2 ? 0 : cur + 1;
    }
    mma_settled(dk);
    mma_settled(dv);
    wait_vmcnt<0>();
    __syncthreads();  // the buffers are free: no load is in flight, no wave reads a tile
  }

  // Accumulators: row = key (8*(r/4) + 4*(l/32) + r%4 of the wave's 32), column = d.  Each wave turns its 32 x D block
  // around in LDS (the tiles are done with) and writes whole 16-byte pieces of rows.
  __syncthreads();
  bf16 *const stage = (wave < 2 ? &Qs[0][0] : &Gs[0][0]) + (wave & 1) * 32 * D;
  static_assert(2 * 32 * D <= NBUF * C::kTile, "staging fits the tile buffers");
  auto write_out = [&](f32x16 const (&acc)[D / 32], float factor, bf16 *out, int64_t row_stride, int dim) {
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        VecIO<bf16>::store1(stage + (8 * (r >> 2) + 4 * h32 + (r & 3)) * D + i * 32 + (lane & 31), acc[i][r] * factor);
    // LDS operations of one wave complete in order: the reads below see the writes above
#pragma unroll
    for (int k = 0; k < 32 * (D / 8) / 64; k++) {
      int const c = lane + k * 64;
      int const row = c / (D / 8), ch = c % (D / 8);
      u32x4 const v = *reinterpret_cast<u32x4 const *>(stage + row * D + ch * 8);
      if (wkv0 + row < p.Skv && (!PAD || ch * 8 < dim)) *reinterpret_cast<u32x4 *>(out + (int64_t)(wkv0 + row) * row_stride + ch * 8) = v;
    }
  };
  write_out(dk, p.grad_scale, static_cast<bf16 *>(p.dk) + (int64_t)b * p.k_bs + (int64_t)kh * dim_qk, p.k_ss, dim_qk);
  write_out(dv, 1.0f, static_cast<bf16 *>(p.dv) + (int64_t)b * p.v_bs + (int64_t)kh * dim_v, p.v_ss, dim_v);
}

template <int D, bool PAD>
static void launch(hipStream_t st, MaskedAttnParams const &p) {
  dim3 const grid((unsigned)(ceil_div(p.Skv, 128) * p.KH * p.B));
  bool const cap = p.capped != 0, bias = p.slopes != nullptr;
  if (cap && bias) masked_dkdv_heads_kernel<D, PAD, true, true><<<grid, 256, 0, st>>>(p);
  else if (cap) masked_dkdv_heads_kernel<D, PAD, true, false><<<grid, 256, 0, st>>>(p);
  else if (bias) masked_dkdv_heads_kernel<D, PAD, false, true><<<grid, 256, 0, st>>>(p);
  else masked_dkdv_heads_kernel<D, PAD, false, false><<<grid, 256, 0, st>>>(p);
}

hipError_t masked_attention_dkdv_heads(hipStream_t st, MaskedAttnParams const &p) {
  if (p.Dq == p.Dv && p.Dq == 64) launch<64, false>(st, p);
  else if (p.Dq == p.Dv && p.Dq == 128) launch<128, false>(st, p);
  else if (p.Dq <= 64 && p.Dv <= 64) launch<64, true>(st, p);
  else launch<128, true>(st, p);
  return hipGetLastError();
}

}  // namespace ffk
