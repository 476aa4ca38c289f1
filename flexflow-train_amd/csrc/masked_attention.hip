// Masked attention: entry points, the rules that choose kernels, the ranges of keys from documents and prefixes, and
// the sum over parts of the keys (see masked_attention.h).
#include "masked_attention.h"
#include <math.h>

namespace ffk {

// instances: masked_attention_{fwd,dq,dkdv}_{bf16,f32}.hip
hipError_t masked_attention_fwd_bf16(hipStream_t st, MaskedAttnParams const &p, int padded, int groups);
hipError_t masked_attention_fwd_f32(hipStream_t st, MaskedAttnParams const &p, int padded, int groups);
hipError_t masked_attention_dq_bf16(hipStream_t st, MaskedAttnParams const &p, int padded, int groups);
hipError_t masked_attention_dq_f32(hipStream_t st, MaskedAttnParams const &p, int padded, int groups);
hipError_t masked_attention_dkdv_bf16(hipStream_t st, MaskedAttnParams const &p, int padded, int groups);
hipError_t masked_attention_dkdv_f32(hipStream_t st, MaskedAttnParams const &p, int padded, int groups);
// bf16 heads up to 128 (heads_kernels below): masked_attention_heads_{fwd,rows,dq,dkdv}.hip
hipError_t masked_attention_fwd_heads(hipStream_t st, MaskedAttnParams const &p);
hipError_t masked_attention_fwd_rows(hipStream_t st, MaskedAttnParams const &p);  // few rows
hipError_t masked_attention_dq_heads(hipStream_t st, MaskedAttnParams const &p);
hipError_t masked_attention_dkdv_heads(hipStream_t st, MaskedAttnParams const &p);

// --------------------------------------------------------------------------
// key ranges
// --------------------------------------------------------------------------
constexpr int kRangeThreads = 256;

// One thread a row: the last document that begins at or before the row's position, by bisection over the starts.  Every
// index stays inside the starts whatever they hold, and the result inside [0, seq_kv].  Bound by the latency of the
// bisection's reads: 64 x 16384 rows, 50 documents, 7.0 us (8 MB written).
__global__ __launch_bounds__(kRangeThreads) void key_ranges_kernel(int2 *out, int const *starts, int const *prefixes, int64_t rows,
                                                                   FastDiv seq_q, int seq_kv, int docs, int causal, int offset) {
  int64_t const at = (int64_t)blockIdx.x * kRangeThreads + threadIdx.x;
  if (at >= rows) return;
  uint32_t b, i;
  seq_q.divmod((uint32_t)at, b, i);
  int const position = offset + (int)i;
  int lo = 0, end = seq_kv, doc = 0;
  if (starts != nullptr) {
    int const *s = starts + (int64_t)b * (docs + 1);
    int below = 0, above = docs + 1;  // starts before `below` are at or before the position, those from `above` on behind it
    while (below < above) {
      int const mid = (below + above) >> 1;
      if (s[mid] <= position) below = mid + 1;
      else above = mid;
    }
    doc = below - 1;
    if (doc < 0 || doc >= docs) {
      out[at] = int2{0, 0};
      return;
    }
    lo = min(max(s[doc], 0), seq_kv);
    end = min(max(s[doc + 1], 0), seq_kv);
  }
  int hi = end;
  if (causal) {
    int const prefix = prefixes != nullptr ? min(max(prefixes[(int64_t)b * docs + doc], 0), seq_kv) : 0;
    hi = min(end, max(position + 1, lo + prefix));
  }
  out[at] = lo < hi ? int2{lo, hi} : int2{0, 0};
}

// --------------------------------------------------------------------------
// the parts of the keys, added up
// --------------------------------------------------------------------------
// One wave a row.  First the lanes are parts, 64 at a time, for the reference point; then they are columns, up to 4 each
// (head sizes to 256), and take the parts' rows eight at a time, so that their loads are in flight together.
template <typename T>
__global__ __launch_bounds__(64) void masked_merge_kernel(MaskedAttnParams p) {
  int const lane = threadIdx.x;
  int64_t const rows = (int64_t)p.B * p.KH * p.R, at = blockIdx.x;
  int const row = (int)(at % p.R), hb = (int)(at / p.R);
  int const kh = hb % p.KH, b = hb / p.KH;
  int i, g;
  row_of(p, row, i, g);
  int const head = kh * p.G + g;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, p.part_ml[2 * (s * rows + at)]);
  m = wave_max(m);
  float const m_use = m == -INFINITY ? 0.0f : m;
  int const d = lane * 4;
  float l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < p.splits; s0 += 64) {
    float f = 0.0f;
    if (s0 + lane < p.splits) {
      float const *ml = p.part_ml + 2 * ((s0 + lane) * rows + at);
      f = __builtin_amdgcn_exp2f(ml[0] - m_use);
      l += ml[1] * f;
    }
    int const n = min(64, p.splits - s0);
    float const *po = p.part_o + (s0 * rows + at) * p.Dv + (d < p.Dv ? d : 0);
    for (int s = 0; s < n; s += 8) {
      f32x4 x[8];
#pragma unroll
      for (int u = 0; u < 8; u++) x[u] = *reinterpret_cast<f32x4 const *>(po + min(s + u, n - 1) * rows * p.Dv);
#pragma unroll
      for (int u = 0; u < 8; u++) {
        // past the last part the last is there again, times 0 (its values are finite, or the row's are not)
        float const fu = s + u < n ? __shfl(f, s + u, 64) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += x[u][e] * fu;
      }
    }
  }
  l = wave_sum(l);
  float const inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (d < p.Dv)
    store4(static_cast<T *>(p.o) + (int64_t)b * p.o_bs + (int64_t)i * p.o_ss + (int64_t)head * p.Dv + d, o[0] * inv, o[1] * inv, o[2] * inv,
           o[3] * inv);
  if (lane == 0 && p.lse != nullptr)
    p.lse[((int64_t)b * p.H + head) * p.Sq + i] = l == 0.0f ? -INFINITY : (m + p.shift + __log2f(l)) * kLn2;
}

// --------------------------------------------------------------------------
// rules
// --------------------------------------------------------------------------
static int padded_head(ffk_masked_attention_desc_t const *d) {
  int64_t const dv = d->v_head_dim != 0 ? d->v_head_dim : d->head_dim;
  int64_t const most = d->head_dim > dv ? d->head_dim : dv;
  return most <= 64 ? 64 : most <= 96 ? 96 : most <= 128 ? 128 : 256;
}
static int64_t rows_of(ffk_masked_attention_desc_t const *d) { return d->seq_q * (d->heads / d->kv_heads); }

static bool heads_kernels(ffk_masked_attention_desc_t const *d, int dtype);
static bool logistic_cap(ffk_masked_attention_desc_t const *d, int dtype) { return dtype == FFK_BF16 && d->score_cap <= kLogisticCap; }
// Workgroups of 128 rows or keys below which those of 32, whose four waves share out the other axis, are better.  fp32, bound
// by its products: as many as CUs (two sequences of 1000 tokens, 8 heads of 64 on 4, causal, 128 workgroups: forward 87 us, and
// 38 with 32 rows, backward 219 and 153; four sequences, 256 workgroups, not causal, 86 and 116, 285 and 367).  bf16: half as
// many (two sequences, 8 heads of 128, 128 workgroups, forward 26 us and 37, backward 75 and 80; 8 heads of 256 on 4, 160
// workgroups, forward 54 and 73; one sequence, 4 heads of 128 on 2, 32 workgroups, forward 25 and 21, backward 99 and 86).
//   Rows over a longer cache are where this is wrong in fp32, whose keys come in parts for either: 16, 32, 64, 128 and 256 rows of
// 32 heads of 128 on 8 over 8192 keys, forward, 42, 76, 125, 230 and 449 us, and 86, 89, 92, 155 and 289 with 128 rows to a
// workgroup.  In bf16 (32 rows in one wave, in parts, or 128 and whole keys) 20, 29, 54, 84 and 122 us, and 158 to 161.
static int few_workgroups(int dtype) { return dtype == FFK_FLOAT ? kNumCU : kNumCU / 2; }
// (FFK_OPTION_ATTENTION_VARIANT other than 0 keeps the kernels for many rows and keys at every size.)
// 32-row groups of a workgroup: 4, or 1 whose four waves share out the keys, where there are no more rows or few
// workgroups.  (fp32 heads past 128 have no such kernel.)
static int row_groups(ffk_masked_attention_desc_t const *d, int dtype) {
  if (dtype == FFK_FLOAT && padded_head(d) > 128) return 4;
  int64_t const rows = rows_of(d);
  if (option(FFK_OPTION_ATTENTION_VARIANT) != 0) return 4;
  return rows <= 32 || ceil_div(rows, 128) * d->kv_heads * d->batch < few_workgroups(dtype) ? 1 : 4;
}
// Parts of the keys, each a workgroup of its own, where few workgroups would run over long keys.  In the kernel of one
// wave a workgroup (masked_attention_heads_rows.hip) ten waves for every CU, each with 256 keys at least: twice what runs at
// a time, so that sequences of several lengths even out (16 of 4096 to 8192 keys, 8 key heads of 128: 86 us, with five 90);
// in the general one two workgroups for every CU, each with 512.
static int key_splits(ffk_masked_attention_desc_t const *d, int dtype) {
  int const groups = row_groups(d, dtype);
  bool const rows_kernel = groups == 1 && heads_kernels(d, dtype);
  if (groups == 4 && heads_kernels(d, dtype)) return 1;  // (masked_attention_heads_fwd.hip takes its keys whole)
  int64_t const workgroups = ceil_div(rows_of(d), 32 * groups) * d->kv_heads * d->batch;
  int64_t const most = d->seq_kv / (rows_kernel ? 256 : 512), enough = rows_kernel ? 10 * kNumCU : 2 * kNumCU;
  if (2 * workgroups > enough || most <= 1) return 1;
  int64_t const want = enough / workgroups;
  return (int)(want < most ? want : most);
}
static size_t split_bytes(ffk_masked_attention_desc_t const *d, int splits) {
  int64_t const dv = d->v_head_dim != 0 ? d->v_head_dim : d->head_dim;
  return splits <= 1 ? 0 : (size_t)splits * d->batch * d->kv_heads * rows_of(d) * (dv + 2) * sizeof(float);
}

static int key_groups(ffk_masked_attention_desc_t const *d, int dtype);
// Whether every launch has fewer than the 2^32 threads that the runtime takes.  (Parts of the keys multiply few workgroups only.)
static bool launches_fit(ffk_masked_attention_desc_t const *d, int dtype, bool backward) {
  int64_t const places = d->kv_heads * d->batch, lim = (int64_t)1 << 32;
  int const groups = row_groups(d, dtype), threads = !backward && groups == 1 && heads_kernels(d, dtype) ? 64 : 256;
  auto const fits = [&](int64_t tiles, int threads) { return tiles * places < lim / threads; };  // (below 2^25 and 2^30)
  return fits(ceil_div(rows_of(d), 32 * groups), threads) && (!backward || fits(ceil_div(d->seq_kv, 32 * key_groups(d, dtype)), 256));
}

static int check(char const *who, int dtype, ffk_masked_attention_desc_t const *d, bool backward) {
  FFK_REQUIRE(d != nullptr, "%s: NULL descriptor", who);
  FFK_REQUIRE(dtype == FFK_BF16 || dtype == FFK_FLOAT, "%s: dtype %d not supported (the entry point takes FLOAT or BF16)", who, dtype);
  FFK_REQUIRE(d->batch > 0 && d->heads > 0 && d->kv_heads > 0 && d->seq_q > 0 && d->seq_kv > 0, "%s: bad shape", who);
  FFK_REQUIRE(d->heads % d->kv_heads == 0, "%s: heads (%lld) must be a multiple of kv_heads (%lld)", who, (long long)d->heads, (long long)d->kv_heads);
  int64_t const unit = dtype == FFK_BF16 ? 8 : 4, dv = d->v_head_dim != 0 ? d->v_head_dim : d->head_dim;
  FFK_REQUIRE(d->head_dim > 0 && dv > 0 && d->head_dim <= 256 && dv <= 256 && d->head_dim % unit == 0 && dv % unit == 0,
              "%s: head sizes must be multiples of %d up to 256", who, (int)unit);
  int64_t const lim = (int64_t)1 << 30;
  FFK_REQUIRE(d->batch < lim && d->heads < lim && d->seq_q < lim && d->seq_kv < lim && d->query_offset >= 0 && d->query_offset < lim,
              "%s: sizes must be below 2^30", who);
  FFK_REQUIRE(rows_of(d) < lim, "%s: seq_q * heads / kv_heads must be below 2^30", who);
  FFK_REQUIRE(d->batch * d->heads < lim, "%s: batch * heads must be below 2^30", who);
  FFK_REQUIRE(d->q_seq_stride % unit == 0 && d->k_seq_stride % unit == 0 && d->v_seq_stride % unit == 0 && d->o_seq_stride % unit == 0 &&
                  d->q_batch_stride % unit == 0 && d->k_batch_stride % unit == 0 && d->v_batch_stride % unit == 0 && d->o_batch_stride % unit == 0,
              "%s: strides must be multiples of %d elements", who, (int)unit);
  int64_t const qw = d->heads * d->head_dim, kw = d->kv_heads * d->head_dim, vw = d->kv_heads * dv, ow = d->heads * dv;
  FFK_REQUIRE(d->q_seq_stride >= qw && d->k_seq_stride >= kw && d->v_seq_stride >= vw && d->o_seq_stride >= ow,
              "%s: a sequence stride is smaller than its row of heads", who);
  FFK_REQUIRE(d->batch == 1 || (d->q_batch_stride >= qw && d->k_batch_stride >= kw && d->v_batch_stride >= vw && d->o_batch_stride >= ow),
              "%s: a batch stride is smaller than a row of heads", who);
  FFK_REQUIRE(d->scale > 0.0f && isfinite(d->scale), "%s: scale must be positive and finite", who);
  FFK_REQUIRE(d->score_cap >= 0.0f && isfinite(d->score_cap) && (d->score_cap == 0.0f || (isfinite(d->scale / d->score_cap * 4.0f) && isfinite(d->score_cap * 4.0f))),
              "%s: score_cap must be 0 (none) or positive, finite and not vanishing beside scale", who);
  FFK_REQUIRE(launches_fit(d, dtype, backward), "%s: too many workgroups", who);
  return FFK_OK;
}

// Biases are added in units of the raw product, or of the cap's tanh (slope_unit): one of up to 2^27 has to be a number there.
static int check_slopes(char const *who, MaskedAttnParams const &p) {
  FFK_REQUIRE(p.slopes == nullptr || p.slope_unit < 0x1p100f, "%s: scale, or score_cap, vanishes beside distance slopes", who);
  return FFK_OK;
}

static MaskedAttnParams params_of(ffk_masked_attention_desc_t const *d, int dtype, void const *q, void const *k, void const *v, int32_t const *ranges,
                                  float const *slopes) {
  MaskedAttnParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.ranges = ranges;
  p.slopes = slopes;
  p.B = (int)d->batch;
  p.H = (int)d->heads;
  p.KH = (int)d->kv_heads;
  p.G = p.H / p.KH;
  p.Sq = (int)d->seq_q;
  p.Skv = (int)d->seq_kv;
  p.Dq = (int)d->head_dim;
  p.Dv = (int)(d->v_head_dim != 0 ? d->v_head_dim : d->head_dim);
  p.R = (int)rows_of(d);
  p.q_bs = d->q_batch_stride; p.q_ss = d->q_seq_stride;
  p.k_bs = d->k_batch_stride; p.k_ss = d->k_seq_stride;
  p.v_bs = d->v_batch_stride; p.v_ss = d->v_seq_stride;
  p.o_bs = d->o_batch_stride; p.o_ss = d->o_seq_stride;
  p.q_offset = (int)d->query_offset;
  p.capped = d->score_cap == 0.0f ? kNoCap : logistic_cap(d, dtype) ? kCapLogistic : kCapTanh;
  p.score_scale = d->scale * kLog2e;
  p.grad_scale = d->scale;
  if (p.capped == kCapLogistic) {
    p.cap_in = -2.0f * kLog2e * (d->scale / d->score_cap);
    p.score_scale = 2.0f * kLog2e * d->score_cap;
    p.shift = -kLog2e * d->score_cap;
    p.grad_scale = 4.0f * d->scale;
  } else if (p.capped == kCapTanh) {
    p.cap_in = d->scale / d->score_cap;
    p.score_scale = kLog2e * d->score_cap;
  }
  p.slope_unit = kLog2e / p.score_scale;
  p.causal = d->causal != 0;
  p.padded_rows = (p.R + 63) / 64 * 64;
  p.group = make_fast_div((uint32_t)p.G);
  p.heads_div = make_fast_div((uint32_t)p.KH);
  p.places_div = make_fast_div((uint32_t)(p.KH * p.B));
  p.splits = 1;
  return p;
}

// The backward's scratch: what the dQ kernels leave of the rows, and the summaries of their ranges.
static size_t row_bytes(ffk_masked_attention_desc_t const *d) {
  return (size_t)d->batch * d->kv_heads * kRowFields * (size_t)(ceil_div(rows_of(d), 64) * 64) * sizeof(float);
}
static size_t backward_bytes(ffk_masked_attention_desc_t const *d) {
  return row_bytes(d) + (size_t)d->batch * ceil_div(rows_of(d), 32) * sizeof(RangeSummary);
}

// The kernels of masked_attention_heads_*.hip: bf16, head sizes up to 128 (64 and 128 themselves, others made longer with
// zeros), no cap or one by the logistic function, rows that byte offsets below 2^31 reach (of all rows of an entry in the dK/dV
// kernel, of a tile in the others).
static bool heads_kernels(ffk_masked_attention_desc_t const *d, int dtype) {
  int64_t const lim = (int64_t)1 << 31;
  return dtype == FFK_BF16 && padded_head(d) <= 128 && logistic_cap(d, dtype) && d->k_seq_stride < (1 << 24) && d->v_seq_stride < (1 << 24) &&
         d->seq_q * d->q_seq_stride * 2 < lim && d->seq_q * d->o_seq_stride * 2 < lim;
}
// 32-key groups of a workgroup of the general dK/dV kernel, and whether it is to run in place of the one for heads: 4, or 1
// whose four waves share out the rows, where there are few workgroups.
static int key_groups(ffk_masked_attention_desc_t const *d, int dtype) {
  if (padded_head(d) > 128) return 4;  // (no registers left for the rows' tiles)
  if (option(FFK_OPTION_ATTENTION_VARIANT) != 0) return 4;
  return rows_of(d) > 32 && ceil_div(d->seq_kv, 128) * d->kv_heads * d->batch < few_workgroups(dtype) ? 1 : 4;
}

}  // namespace ffk

using namespace ffk;

extern "C" int ffk_attention_key_ranges(ffk_stream_t stream, int64_t batch, int64_t seq_q, int64_t seq_kv, int64_t query_offset, int causal,
                                        int32_t const *document_starts, int64_t num_documents, int32_t const *prefix_lengths,
                                        int32_t *key_ranges) {
  int64_t const lim = (int64_t)1 << 30;
  FFK_REQUIRE(batch > 0 && seq_q > 0 && seq_kv > 0, "attention_key_ranges: bad shape");
  FFK_REQUIRE(batch < lim && seq_q < lim && seq_kv < lim && query_offset >= 0 && query_offset < lim && batch * seq_q < 2 * lim,
              "attention_key_ranges: sizes must be below 2^30, batch * seq_q below 2^31");
  FFK_REQUIRE(key_ranges != nullptr && reinterpret_cast<uintptr_t>(key_ranges) % 8 == 0,
              "attention_key_ranges: key_ranges must be given, 8-byte aligned");
  FFK_REQUIRE(document_starts == nullptr ? num_documents <= 1 : num_documents >= 1 && num_documents < lim,
              "attention_key_ranges: num_documents (%lld) does not fit document_starts", (long long)num_documents);
  FFK_REQUIRE(prefix_lengths == nullptr || causal, "attention_key_ranges: a prefix says nothing without a causal mask");
  int const docs = document_starts != nullptr ? (int)num_documents : 1;
  int64_t const rows = batch * seq_q;
  key_ranges_kernel<<<dim3((unsigned)ceil_div(rows, kRangeThreads)), kRangeThreads, 0, as_stream(stream)>>>(
      reinterpret_cast<int2 *>(key_ranges), document_starts, prefix_lengths, rows, make_fast_div((uint32_t)seq_q), (int)seq_kv, docs, causal,
      (int)query_offset);
  FFK_CHECK_LAUNCH();
  return FFK_OK;
}

extern "C" size_t ffk_masked_attention_forward_workspace_bytes(ffk_masked_attention_desc_t const *d, int dtype) {
  if (check("masked_attention_forward", dtype, d, false) != FFK_OK) return 0;
  return split_bytes(d, key_splits(d, dtype));
}

extern "C" int ffk_masked_attention_forward(ffk_stream_t stream, int dtype, ffk_masked_attention_desc_t const *d, void const *q,
                                            void const *k, void const *v, int32_t const *key_ranges, float const *distance_slopes,
                                            void *o, float *lse, void *workspace, size_t workspace_bytes) {
  int const rc = check("masked_attention_forward", dtype, d, false);
  if (rc != FFK_OK) return rc;
  FFK_REQUIRE(q && k && v && o, "masked_attention_forward: NULL tensor");
  FFK_REQUIRE(o != q && o != k && o != v, "masked_attention_forward: the output is an input");
  FFK_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o), "masked_attention_forward: tensors must be 16-byte aligned");
  FFK_REQUIRE(reinterpret_cast<uintptr_t>(key_ranges) % 8 == 0, "masked_attention_forward: key_ranges must be 8-byte aligned");
  MaskedAttnParams p = params_of(d, dtype, q, k, v, key_ranges, distance_slopes);
  if (int const bad = check_slopes("masked_attention_forward", p)) return bad;
  p.o = o;
  p.lse = lse;
  hipStream_t const st = as_stream(stream);
  int const splits = key_splits(d, dtype);
  if (splits > 1 && workspace != nullptr && aligned16(workspace) && workspace_bytes >= split_bytes(d, splits)) {
    p.splits = splits;
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = p.part_o + (int64_t)splits * p.B * p.KH * p.R * p.Dv;
  }
  int const groups = row_groups(d, dtype);
  auto const general = dtype == FFK_BF16 ? masked_attention_fwd_bf16 : masked_attention_fwd_f32;
  if (!heads_kernels(d, dtype)) FFK_HIP(general(st, p, padded_head(d), groups));
  else if (groups == 4) FFK_HIP(masked_attention_fwd_heads(st, p));
  else FFK_HIP(masked_attention_fwd_rows(st, p));
  if (p.splits > 1) {
    dim3 const grid((unsigned)((int64_t)p.B * p.KH * p.R));
    if (dtype == FFK_BF16) masked_merge_kernel<bf16><<<grid, 64, 0, st>>>(p);
    else masked_merge_kernel<float><<<grid, 64, 0, st>>>(p);
    FFK_CHECK_LAUNCH();
  }
  return FFK_OK;
}

extern "C" size_t ffk_masked_attention_backward_workspace_bytes(ffk_masked_attention_desc_t const *d, int dtype) {
  if (check("masked_attention_backward", dtype, d, true) != FFK_OK) return 0;
  return backward_bytes(d);
}

extern "C" int ffk_masked_attention_backward(ffk_stream_t stream, int dtype, ffk_masked_attention_desc_t const *d, void const *q,
                                             void const *k, void const *v, int32_t const *key_ranges, float const *distance_slopes,
                                             void const *o, void const *d_o, float const *lse, void *dq, void *dk, void *dv,
                                             void *workspace, size_t workspace_bytes) {
  int const rc = check("masked_attention_backward", dtype, d, true);
  if (rc != FFK_OK) return rc;
  FFK_REQUIRE(q && k && v && o && d_o && lse && dq && dk && dv, "masked_attention_backward: NULL tensor");
  // (the dK/dV kernel reads all inputs behind the dQ kernel)
  for (void const *grad : {dq, dk, dv})
    FFK_REQUIRE(grad != q && grad != k && grad != v && grad != o && grad != d_o, "masked_attention_backward: a gradient is an input");
  FFK_REQUIRE(dq != dk && dq != dv && dk != dv, "masked_attention_backward: two gradients are one");
  FFK_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(d_o) && aligned16(dq) && aligned16(dk) && aligned16(dv),
              "masked_attention_backward: tensors must be 16-byte aligned");
  FFK_REQUIRE(reinterpret_cast<uintptr_t>(key_ranges) % 8 == 0, "masked_attention_backward: key_ranges must be 8-byte aligned");
  size_t const need = backward_bytes(d);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need) {
    return fail(FFK_ERR_WORKSPACE, "masked_attention_backward: workspace must hold %zu bytes, 16-byte aligned (%zu given)", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  }
  MaskedAttnParams p = params_of(d, dtype, q, k, v, key_ranges, distance_slopes);
  if (int const bad = check_slopes("masked_attention_backward", p)) return bad;
  p.o = const_cast<void *>(o);
  p.d_o = d_o;
  p.lse = const_cast<float *>(lse);
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.rows = static_cast<float *>(workspace);
  p.summary = reinterpret_cast<RangeSummary *>(static_cast<uint8_t *>(workspace) + row_bytes(d));
  hipStream_t const st = as_stream(stream);
  int const padded = padded_head(d);
  auto const launch_dq = dtype == FFK_BF16 ? masked_attention_dq_bf16 : masked_attention_dq_f32;
  auto const launch_dkdv = dtype == FFK_BF16 ? masked_attention_dkdv_bf16 : masked_attention_dkdv_f32;
  int const groups = row_groups(d, dtype);
  if (groups == 4 && heads_kernels(d, dtype)) FFK_HIP(masked_attention_dq_heads(st, p));
  else FFK_HIP(launch_dq(st, p, padded, groups));
  int const keys = key_groups(d, dtype);
  if (keys == 4 && heads_kernels(d, dtype)) FFK_HIP(masked_attention_dkdv_heads(st, p));
  else FFK_HIP(launch_dkdv(st, p, padded, keys));
  return FFK_OK;
}
