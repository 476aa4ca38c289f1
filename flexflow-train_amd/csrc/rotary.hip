// Rotary positions with up to four axes, forward and backward, for gfx950.
//
// Column pair j of a head (j and j + n/2 of the first n columns, or 2j and 2j + 1) turns by the angle
// theta = position of the token on the pair's axis * frequency_j:
//   (a, b) -> (a cos theta - b sin theta, a sin theta + b cos theta);
// the gradient turns back by -theta.  Columns from n on pass through.
//
// The angles of a token are the same for all heads: a workgroup takes a few tokens, computes their cosines and sines
// once into LDS and turns all heads of q and k with them.  The product position * frequency is taken in 64 bits and
// brought into one turn there, so that far positions keep fp32 accuracy of the angle (in 32 bits position 10^6 has lost
// 20 of its 24 bits).  Bound by memory: every element is read and written once (bf16, 4 x 4096 tokens, 40 heads of 128:
// 64 us, 5.2 TB/s; fp32, 2 x 196 tokens, 24 heads of 64: 3.8 us, launch latency).
#include "ffk_common.h"
#include <math.h>

namespace ffk {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPairs = 2048;  // pairs a workgroup has room for in LDS

struct RotaryTensor {
  void const *in;
  void *out;
  int64_t in_bs, in_ss, out_bs, out_ss;
  int heads;
};
struct RotaryParams {
  RotaryTensor t[2];
  int const *positions;  // [axes, batch, seq]
  float const *frequencies;
  int64_t tokens;
  int seq, head_dim, half, tokens_per_wg;
  int section_end[4];  // pair j belongs to the first axis with j < section_end
  float sign;
  FastDiv seq_div, half_div;
  FastDiv units_div;  // units of a head
  int units, turning;  // of a head: all, and those that turn
  FastDiv heads_div;   // heads of q and k together
  int heads;
};

// N elements as floats, any N of 1, 2, 4, 8 with N * sizeof(T) <= 16
template <typename T, int N>
__device__ __forceinline__ void load_some(T const *p, float (&v)[N]) {
  if constexpr (N * sizeof(T) == 16) {
    VecIO<T>::load(p, v);
  } else if constexpr (sizeof(T) == 4) {
    if constexpr (N == 2) {
      f32x2 const r = *reinterpret_cast<f32x2 const *>(p);
      v[0] = r[0];
      v[1] = r[1];
    } else {
      v[0] = *p;
    }
  } else if constexpr (N == 4) {
    u32x2 const r = *reinterpret_cast<u32x2 const *>(p);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  } else if constexpr (N == 2) {
    uint32_t const r = *reinterpret_cast<uint32_t const *>(p);
    v[0] = __uint_as_float(r << 16);
    v[1] = __uint_as_float(r & 0xffff0000u);
  } else {
    v[0] = VecIO<T>::load1(p);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_some(T *p, float const (&v)[N]) {
  if constexpr (N * sizeof(T) == 16) {
    VecIO<T>::store(p, v);
  } else if constexpr (sizeof(T) == 4) {
    if constexpr (N == 2) *reinterpret_cast<f32x2 *>(p) = f32x2{v[0], v[1]};
    else *p = v[0];
  } else if constexpr (N == 4) {
    *reinterpret_cast<u32x2 *>(p) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint32_t *>(p) = pack_bf16x2(v[0], v[1]);
  } else {
    VecIO<T>::store1(p, v[0]);
  }
}

// A unit: halves apart, N elements of the first half and the N of the second that they turn with; interleaved, the N / 2 pairs
// of N elements in a row, so that a wave's accesses follow each other (two accesses of N to a unit, which leave gaps between
// lanes: fp32, 7 x 561 tokens, 60 heads of 128, 60 us and 47).  (N = 1 interleaved: two single elements.)
template <typename T, int N, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryParams p) {
  __shared__ float cosines[kRotaryPairs], sines[kRotaryPairs];
  int64_t const token0 = (int64_t)blockIdx.x * p.tokens_per_wg;
  int const tokens = (int)min((int64_t)p.tokens_per_wg, p.tokens - token0);
  for (int i = threadIdx.x; i < tokens * p.half; i += kRotaryThreads) {
    uint32_t tk, j;
    p.half_div.divmod((uint32_t)i, tk, j);
    int const axis = ((int)j >= p.section_end[0]) + ((int)j >= p.section_end[1]) + ((int)j >= p.section_end[2]);
    int const position = p.positions[axis * p.tokens + token0 + tk];
    double turns = (double)position * (double)p.frequencies[j] * 0.15915494309189533577;
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    cosines[i] = c;
    sines[i] = s * p.sign;
  }
  __syncthreads();
  int const all = tokens * p.heads * p.units;
  for (int i = threadIdx.x; i < all; i += kRotaryThreads) {
    uint32_t rest, unit, tk, head;
    p.units_div.divmod((uint32_t)i, rest, unit);
    p.heads_div.divmod(rest, tk, head);
    uint32_t b, s;
    p.seq_div.divmod((uint32_t)(token0 + tk), b, s);
    bool const is_k = (int)head >= p.t[0].heads;
    int const h = is_k ? (int)head - p.t[0].heads : (int)head;
    T const *in = static_cast<T const *>(is_k ? p.t[1].in : p.t[0].in) + (int64_t)b * (is_k ? p.t[1].in_bs : p.t[0].in_bs) +
                  (int64_t)s * (is_k ? p.t[1].in_ss : p.t[0].in_ss) + (int64_t)h * p.head_dim;
    T *out = static_cast<T *>(is_k ? p.t[1].out : p.t[0].out) + (int64_t)b * (is_k ? p.t[1].out_bs : p.t[0].out_bs) +
             (int64_t)s * (is_k ? p.t[1].out_ss : p.t[0].out_ss) + (int64_t)h * p.head_dim;
    float x[N], y[N];
    if (INTERLEAVED && N > 1 && (int)unit < p.turning) {
      int const j = (int)unit * (N / 2);
      load_some<T, N>(in + 2 * j, x);
      float const *cs = cosines + tk * p.half + j, *sn = sines + tk * p.half + j;
#pragma unroll
      for (int e = 0; e < N / 2; e++) {
        float const a = x[2 * e], bb = x[2 * e + 1];
        x[2 * e] = a * cs[e] - bb * sn[e];
        x[2 * e + 1] = a * sn[e] + bb * cs[e];
      }
      store_some<T, N>(out + 2 * j, x);
    } else if ((int)unit < p.turning) {
      int const j = (int)unit * N;
      int const at_a = INTERLEAVED ? 2 * j : j, at_b = INTERLEAVED ? 2 * j + 1 : j + p.half;
      load_some<T, N>(in + at_a, x);
      load_some<T, N>(in + at_b, y);
      float const *cs = cosines + tk * p.half + j, *sn = sines + tk * p.half + j;
#pragma unroll
      for (int e = 0; e < N; e++) {
        float const a = x[e], bb = y[e];
        x[e] = a * cs[e] - bb * sn[e];
        y[e] = a * sn[e] + bb * cs[e];
      }
      store_some<T, N>(out + at_a, x);
      store_some<T, N>(out + at_b, y);
    } else {
      // columns that pass through, N at a time
      int const at = 2 * p.half + ((int)unit - p.turning) * N;
      load_some<T, N>(in + at, x);
      store_some<T, N>(out + at, x);
    }
  }
}

template <typename T, int N>
static int rotary_launch(char const *who, hipStream_t st, RotaryParams &p, bool interleaved, bool copy_rest) {
  p.turning = interleaved && N > 1 ? 2 * p.half / N : p.half / N;
  p.units = p.turning + (copy_rest ? (p.head_dim - 2 * p.half) / N : 0);
  p.units_div = make_fast_div((uint32_t)p.units);
  // as many tokens as give every thread a few units, while every CU has workgroups
  int64_t const per_token = (int64_t)p.heads * p.units;
  int64_t want = ceil_div(4 * kRotaryThreads, per_token);
  int64_t const even = ceil_div(p.tokens, 4 * kNumCU), room = kRotaryPairs / p.half;
  if (want > even) want = even;
  if (want > room) want = room;
  if (want < 1) want = 1;
  p.tokens_per_wg = (int)want;
  // (2^32 threads are more than a launch takes)
  FFK_REQUIRE(ceil_div(p.tokens, want) < ((int64_t)1 << 32) / kRotaryThreads, "%s: too many workgroups (%lld tokens, %lld to each)", who,
              (long long)p.tokens, (long long)want);
  dim3 const grid((unsigned)ceil_div(p.tokens, want));
  if (interleaved) rotary_kernel<T, N, true><<<grid, kRotaryThreads, 0, st>>>(p);
  else rotary_kernel<T, N, false><<<grid, kRotaryThreads, 0, st>>>(p);
  FFK_CHECK_LAUNCH();
  return FFK_OK;
}

static int rotary_any(char const *who, ffk_stream_t stream, int dtype, ffk_rotary_desc_t const *d, void const *q, void const *k,
                      int32_t const *positions, float const *frequencies, void *q_out, void *k_out, float sign) {
  FFK_REQUIRE(d != nullptr, "%s: NULL descriptor", who);
  FFK_REQUIRE(dtype == FFK_BF16 || dtype == FFK_FLOAT, "%s: dtype %d not supported (the entry point takes FLOAT or BF16)", who, dtype);
  FFK_REQUIRE(d->batch > 0 && d->seq > 0 && d->q_heads > 0 && d->k_heads >= 0 && d->head_dim > 0, "%s: bad shape", who);
  int64_t const lim = (int64_t)1 << 30;
  FFK_REQUIRE(d->batch < lim && d->seq < lim && d->batch * d->seq < lim, "%s: batch * seq must be below 2^30", who);
  FFK_REQUIRE(d->num_axes >= 1 && d->num_axes <= 4, "%s: one to four axes, not %lld", who, (long long)d->num_axes);
  int64_t half = 0;
  for (int a = 0; a < d->num_axes; a++) {
    FFK_REQUIRE(d->sections[a] >= 0 && d->sections[a] <= d->head_dim, "%s: bad section %lld", who, (long long)d->sections[a]);
    half += d->sections[a];
  }
  FFK_REQUIRE(half >= 1 && 2 * half <= d->head_dim, "%s: the sections' pairs (%lld) do not fit the head size %lld", who, (long long)half,
              (long long)d->head_dim);
  FFK_REQUIRE(half <= kRotaryPairs && d->head_dim <= 65536 && (d->q_heads + d->k_heads) < 65536 && (d->q_heads + d->k_heads) * d->head_dim < lim,
              "%s: at most %d pairs a head, 65535 heads", who, kRotaryPairs);
  FFK_REQUIRE(q && q_out && positions && frequencies, "%s: NULL tensor", who);
  FFK_REQUIRE(d->k_heads == 0 || (k && k_out), "%s: NULL tensor", who);
  FFK_REQUIRE(d->k_heads == 0 || (q_out != k_out && q_out != k && k_out != q), "%s: an output is the other tensor", who);
  int64_t const qw = d->q_heads * d->head_dim, kw = d->k_heads * d->head_dim;
  FFK_REQUIRE(d->q_seq_stride >= qw && d->q_out_seq_stride >= qw && (d->k_heads == 0 || (d->k_seq_stride >= kw && d->k_out_seq_stride >= kw)),
              "%s: a sequence stride is smaller than its row of heads", who);
  FFK_REQUIRE(d->batch == 1 || (d->q_batch_stride >= qw && d->q_out_batch_stride >= qw &&
                                (d->k_heads == 0 || (d->k_batch_stride >= kw && d->k_out_batch_stride >= kw))),
              "%s: a batch stride is smaller than a row of heads", who);
  bool const q_in_place = q == q_out, k_in_place = d->k_heads == 0 || k == k_out;
  FFK_REQUIRE(!q_in_place || (d->q_seq_stride == d->q_out_seq_stride && (d->batch == 1 || d->q_batch_stride == d->q_out_batch_stride)),
              "%s: in place, input and output have the same strides", who);
  FFK_REQUIRE(d->k_heads == 0 || k != k_out || (d->k_seq_stride == d->k_out_seq_stride && (d->batch == 1 || d->k_batch_stride == d->k_out_batch_stride)),
              "%s: in place, input and output have the same strides", who);
  RotaryParams p = {};
  p.t[0] = RotaryTensor{q, q_out, d->q_batch_stride, d->q_seq_stride, d->q_out_batch_stride, d->q_out_seq_stride, (int)d->q_heads};
  p.t[1] = RotaryTensor{k, k_out, d->k_batch_stride, d->k_seq_stride, d->k_out_batch_stride, d->k_out_seq_stride, (int)d->k_heads};
  p.positions = positions;
  p.frequencies = frequencies;
  p.tokens = d->batch * d->seq;
  p.seq = (int)d->seq;
  p.head_dim = (int)d->head_dim;
  p.half = (int)half;
  int64_t end = 0;
  for (int a = 0; a < 4; a++) {
    if (a < d->num_axes) end += d->sections[a];
    p.section_end[a] = a < d->num_axes - 1 ? (int)end : (int)half;  // the last axis takes what is left
  }
  p.sign = sign;
  p.heads = (int)(d->q_heads + d->k_heads);
  p.seq_div = make_fast_div((uint32_t)d->seq);
  p.half_div = make_fast_div((uint32_t)half);
  p.heads_div = make_fast_div((uint32_t)p.heads);
  // the widest access that every row, both halves and the rest of a head allow
  uint64_t bits = (uint64_t)half | (uint64_t)d->head_dim | (uint64_t)d->q_seq_stride | (uint64_t)d->q_out_seq_stride;
  if (d->batch > 1) bits |= (uint64_t)d->q_batch_stride | (uint64_t)d->q_out_batch_stride;
  uint64_t at = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out);
  if (d->k_heads > 0) {
    bits |= (uint64_t)d->k_seq_stride | (uint64_t)d->k_out_seq_stride;
    if (d->batch > 1) bits |= (uint64_t)d->k_batch_stride | (uint64_t)d->k_out_batch_stride;
    at |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out);
  }
  int const size = (int)dtype_size(dtype);
  FFK_REQUIRE(at % size == 0, "%s: a tensor is not aligned to its elements", who);
  int n = 16 / size;
  while (n > 1 && (bits % n != 0 || at % (uint64_t)(n * size) != 0)) n /= 2;
  bool const copy_rest = (!q_in_place || !k_in_place) && 2 * half < d->head_dim;
  hipStream_t const st = as_stream(stream);
  bool const inter = d->interleaved != 0;
  if (dtype == FFK_BF16) {
    return n == 8   ? rotary_launch<bf16, 8>(who, st, p, inter, copy_rest)
           : n == 4 ? rotary_launch<bf16, 4>(who, st, p, inter, copy_rest)
           : n == 2 ? rotary_launch<bf16, 2>(who, st, p, inter, copy_rest)
                    : rotary_launch<bf16, 1>(who, st, p, inter, copy_rest);
  }
  return n == 4   ? rotary_launch<float, 4>(who, st, p, inter, copy_rest)
         : n == 2 ? rotary_launch<float, 2>(who, st, p, inter, copy_rest)
                  : rotary_launch<float, 1>(who, st, p, inter, copy_rest);
}

}  // namespace ffk

using namespace ffk;

extern "C" int ffk_rotary_forward(ffk_stream_t stream, int dtype, ffk_rotary_desc_t const *desc, void const *q, void const *k,
                                  int32_t const *positions, float const *frequencies, void *q_out, void *k_out) {
  return rotary_any("rotary_forward", stream, dtype, desc, q, k, positions, frequencies, q_out, k_out, 1.0f);
}

extern "C" int ffk_rotary_backward(ffk_stream_t stream, int dtype, ffk_rotary_desc_t const *desc, void const *q_out_grad,
                                   void const *k_out_grad, int32_t const *positions, float const *frequencies, void *q_grad,
                                   void *k_grad) {
  return rotary_any("rotary_backward", stream, dtype, desc, q_out_grad, k_out_grad, positions, frequencies, q_grad, k_grad, -1.0f);
}
