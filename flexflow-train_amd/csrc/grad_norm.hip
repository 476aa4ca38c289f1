// The norm over many gradient tensors as if they were one vector, and the gradients scaled down to a largest norm, for
// gfx950.  (The update kernels of optimizer.hip take gradients as they are.)
//
//   norm = sqrt(sum over all tensors and elements of g^2)        clipped = g * min(1, max_norm / (norm + 1e-6))
//
// All tensors of a launch are cut into pieces of one size, and a fixed number of workgroups takes them in turn, so a list of
// small biases and large matrices costs one launch.  Squares are taken and summed in 64 bits: neither 1e30 nor 1e-30
// leaves the range then, and every sum has a fixed order.  Bound by memory, also with the conversions: the tensors are
// read once for the norm, and once more, and written, for the clipping.
//   For the norm a thousand workgroups take pieces of 32 KB, of large lists by loads that keep nothing in the caches (2.4 GB
// of bf16: 343 us, 7.0 TB/s, and by ordinary ones 422 us; where the clipping finds the list in the caches the ordinary ones are
// better: 50 MB of fp32, norm and clipping 28 us and 30).  For the clipping every piece of 16 KB is a workgroup of its own, which asks
// for its piece first and adds up the norm while that is on its way (2.4 GB: 830 us, 5.8 TB/s; 2048 workgroups that take
// pieces in turn 946 us).
//   Past a table of 96 tensors every workgroup of the clipping reads another 8 KB of sums for each 96: 2.4 GB of bf16 in 54, 300
// and 1200 tensors take 840, 1065 and 1823 us, the norm's launches 351, 368 and 408.
#include "ffk_common.h"
#include <math.h>
#include <algorithm>
#include <memory>
#include <new>

namespace ffk {

constexpr int kNormThreads = 256;
constexpr int kNormWorkgroups = 1024;  // of a launch for the norm, at most: four on every CU
constexpr int kNormTensors = 96;       // of a launch (the table travels as its argument)
constexpr int64_t kNormKept = 128 << 20;  // bytes of a list up to which its tensors are to stay in the caches
constexpr int kNormLoads = 8, kClipLoads = 4;  // 16-byte loads of a thread in a piece
constexpr int64_t kClipPieces = (1 << 24) - 1;  // of a launch for the clipping, each a workgroup: 2^32 threads are too many

// elements of a piece
__host__ __device__ constexpr int piece_elems(int loads, bool is_bf16) { return loads * kNormThreads * (is_bf16 ? 8 : 4); }

struct NormTable {
  void const *in[kNormTensors];
  void *out[kNormTensors];
  int64_t elems[kNormTensors];
  int first_piece[kNormTensors + 1];
  uint8_t is_bf16[kNormTensors];
  int tensors;
};

__device__ __forceinline__ double square_sum(u32x4 r, float const *) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    double const x = (double)__uint_as_float(r[i]);
    s = __builtin_fma(x, x, s);
  }
  return s;
}
__device__ __forceinline__ double square_sum(u32x4 r, bf16 const *) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    double const x = (double)__uint_as_float(r[i] << 16), y = (double)__uint_as_float(r[i] & 0xffff0000u);
    s = __builtin_fma(x, x, s);
    s = __builtin_fma(y, y, s);
  }
  return s;
}

// the tensor that piece `piece` of the launch belongs to
__device__ __forceinline__ int tensor_of(NormTable const &a, int piece) {
  int below = 0, above = a.tensors;  // first_piece[below] <= piece < first_piece[above]
  while (above - below > 1) {
    int const mid = (below + above) >> 1;
    if (a.first_piece[mid] <= piece) below = mid;
    else above = mid;
  }
  return below;
}

// A 16-byte load, of any alignment that an element has, that keeps nothing in the caches.
typedef u32x4 u32x4_by_2 __attribute__((aligned(2), may_alias));
typedef u32x4 u32x4_by_4 __attribute__((aligned(4), may_alias));
__device__ __forceinline__ u32x4 load_raw_once(bf16 const *p) { return __builtin_nontemporal_load(reinterpret_cast<u32x4_by_2 const *>(p)); }
__device__ __forceinline__ u32x4 load_raw_once(float const *p) { return __builtin_nontemporal_load(reinterpret_cast<u32x4_by_4 const *>(p)); }
template <bool ONCE, typename T>
__device__ __forceinline__ double piece_squares(T const *p, int n) {
  constexpr int V = VecIO<T>::kVec;
  double s = 0.0;
  if (n == piece_elems(kNormLoads, sizeof(T) == 2)) {
    u32x4 r[kNormLoads];
#pragma unroll
    for (int k = 0; k < kNormLoads; k++) r[k] = ONCE ? load_raw_once(p + (k * kNormThreads + threadIdx.x) * V) : load_raw_any(p + (k * kNormThreads + threadIdx.x) * V);
#pragma unroll
    for (int k = 0; k < kNormLoads; k++) s += square_sum(r[k], p);
  } else {
    for (int i = threadIdx.x * V; i < n; i += kNormThreads * V)
      s += square_sum(i + V <= n ? load_raw_any(p + i) : load_raw_first(p + i, n - i), p);
  }
  return s;
}

__device__ __forceinline__ double workgroup_sum(double v, double *lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

template <bool ONCE>
__global__ __launch_bounds__(kNormThreads) void square_sum_kernel(NormTable a, double *partial) {
  __shared__ double lds[4];
  double s = 0.0;
  for (int piece = blockIdx.x; piece < a.first_piece[a.tensors]; piece += gridDim.x) {
    int const i = tensor_of(a, piece);
    int const whole = piece_elems(kNormLoads, a.is_bf16[i]);
    int64_t const at = (int64_t)(piece - a.first_piece[i]) * whole;
    int const n = (int)min((int64_t)whole, a.elems[i] - at);
    s += a.is_bf16[i] ? piece_squares<ONCE>(static_cast<bf16 const *>(a.in[i]) + at, n)
                      : piece_squares<ONCE>(static_cast<float const *>(a.in[i]) + at, n);
  }
  s = workgroup_sum(s, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The norm from the workgroups' sums, the same for every workgroup that computes it.
__device__ __forceinline__ double norm_of(double const *partial, int count, double *lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += kNormThreads) s += partial[i];
  return sqrt(workgroup_sum(s, lds));
}

__global__ __launch_bounds__(kNormThreads) void norm_kernel(double const *partial, int count, float *norm) {
  __shared__ double lds[4];
  double const n = norm_of(partial, count, lds);
  if (threadIdx.x == 0) *norm = (float)n;
}

// A whole piece, fetched already, or one that ends earlier.
template <typename T>
__device__ __forceinline__ void piece_scaled(T const *p, T *q, int n, float factor, u32x4 const (&r)[kClipLoads]) {
  constexpr int V = VecIO<T>::kVec;
  float v[V];
  if (n == piece_elems(kClipLoads, sizeof(T) == 2)) {
#pragma unroll
    for (int k = 0; k < kClipLoads; k++) {
      unpack_raw(r[k], v, p);
#pragma unroll
      for (int e = 0; e < V; e++) v[e] *= factor;
      store_raw_any(q + (k * kNormThreads + threadIdx.x) * V, pack_raw(v, p));
    }
  } else {
    for (int i = threadIdx.x * V; i < n; i += kNormThreads * V) {
      bool const whole = i + V <= n;
      unpack_raw(whole ? load_raw_any(p + i) : load_raw_first(p + i, n - i), v, p);
#pragma unroll
      for (int e = 0; e < V; e++) v[e] *= factor;
      if (whole) store_raw_any(q + i, pack_raw(v, p));
      else store_raw_first(q + i, pack_raw(v, p), n - i);
    }
  }
}

// Every workgroup adds up the norm for itself from the partial sums, a thousand for each table, which the caches hold:
// no third launch between the norm and the scaling.  A tensor that stays as it is, in place, is not touched; its pieces are not asked for
// before that is known.
__global__ __launch_bounds__(kNormThreads) void clip_kernel(NormTable a, double const *partial, int count, float max_norm, float *norm) {
  __shared__ double lds[4];
  int const piece = blockIdx.x, i = tensor_of(a, piece);
  bool const is_bf16 = a.is_bf16[i] != 0, in_place = a.in[i] == a.out[i];
  int const whole = piece_elems(kClipLoads, is_bf16);
  int64_t const at = (int64_t)(piece - a.first_piece[i]) * whole;
  int const n = (int)min((int64_t)whole, a.elems[i] - at);
  u32x4 r[kClipLoads];
  auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kClipLoads; k++) {
      int const e = k * kNormThreads + threadIdx.x;
      if (is_bf16) r[k] = load_raw_any(static_cast<bf16 const *>(a.in[i]) + at + e * 8);
      else r[k] = load_raw_any(static_cast<float const *>(a.in[i]) + at + e * 4);
    }
  };
  if (!in_place && n == whole) fetch();
  double const length = norm_of(partial, count, lds);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)length;
  double const f = (double)max_norm / (length + 1e-6);
  float const factor = f >= 1.0 ? 1.0f : (float)f;  // (a norm that is no number makes the gradients none)
  if (in_place) {
    if (factor == 1.0f) return;
    if (n == whole) fetch();
  }
  if (is_bf16) piece_scaled(static_cast<bf16 const *>(a.in[i]) + at, static_cast<bf16 *>(a.out[i]) + at, n, factor, r);
  else piece_scaled(static_cast<float const *>(a.in[i]) + at, static_cast<float *>(a.out[i]) + at, n, factor, r);
}

static int check_list(char const *who, int const *dtypes, void const *const *grads, int64_t const *elems, int num) {
  FFK_REQUIRE(num >= 0, "%s: negative number of tensors", who);
  FFK_REQUIRE(num == 0 || (dtypes != nullptr && grads != nullptr && elems != nullptr), "%s: NULL list", who);
  for (int i = 0; i < num; i++) {
    FFK_REQUIRE(dtypes[i] == FFK_FLOAT || dtypes[i] == FFK_BF16, "%s: dtype %d of tensor %d not supported (FLOAT or BF16)", who, dtypes[i], i);
    FFK_REQUIRE(elems[i] >= 0 && elems[i] <= kClipPieces * piece_elems(kClipLoads, dtypes[i] == FFK_BF16), "%s: bad size of tensor %d", who, i);
    FFK_REQUIRE(elems[i] == 0 || grads[i] != nullptr, "%s: tensor %d is NULL", who, i);
    FFK_REQUIRE(reinterpret_cast<uintptr_t>(grads[i]) % dtype_size(dtypes[i]) == 0, "%s: tensor %d is not aligned to its elements", who, i);
  }
  return FFK_OK;
}

// Whether no output lies on another output or on another tensor's input: the pieces are worked on in no order.
static int check_apart(char const *who, int const *dtypes, void const *const *grads, void *const *clipped, int64_t const *elems, int num) {
  struct Span {
    uintptr_t begin, end;
    bool out;
  };
  std::unique_ptr<Span[]> const spans(new (std::nothrow) Span[2 * (size_t)num]);
  FFK_REQUIRE(num == 0 || spans != nullptr, "%s: no host memory", who);
  int n = 0;
  for (int i = 0; i < num; i++) {
    if (elems[i] == 0) continue;
    uintptr_t const in = reinterpret_cast<uintptr_t>(grads[i]), out = reinterpret_cast<uintptr_t>(clipped[i]);
    uintptr_t const bytes = (uintptr_t)elems[i] * dtype_size(dtypes[i]);
    spans[n++] = Span{out, out + bytes, true};
    if (in != out) spans[n++] = Span{in, in + bytes, false};
  }
  std::sort(spans.get(), spans.get() + n, [](Span const &a, Span const &b) { return a.begin < b.begin; });
  uintptr_t in_end = 0, out_end = 0;
  for (int i = 0; i < n; i++) {
    FFK_REQUIRE(spans[i].begin >= out_end && (!spans[i].out || spans[i].begin >= in_end), "%s: tensors overlap", who);
    uintptr_t &end = spans[i].out ? out_end : in_end;
    if (spans[i].end > end) end = spans[i].end;
  }
  return FFK_OK;
}

// The tensors from `first` on that one launch takes, as its table: of up to `most` pieces, which no tensor has more of.  Returns
// the first that it does not take.
static int fill_table(NormTable &a, int const *dtypes, void const *const *grads, void *const *out, int64_t const *elems, int num, int first,
                      int loads, int64_t most) {
  a.tensors = 0;
  int64_t pieces = 0;
  int i = first;
  for (; i < num && a.tensors < kNormTensors; i++) {
    if (elems[i] == 0) continue;
    int64_t const more = ceil_div(elems[i], piece_elems(loads, dtypes[i] == FFK_BF16));
    if (pieces + more > most) break;
    int const t = a.tensors++;
    a.in[t] = grads[i];
    a.out[t] = out != nullptr ? out[i] : nullptr;
    a.elems[t] = elems[i];
    a.is_bf16[t] = dtypes[i] == FFK_BF16;
    a.first_piece[t] = (int)pieces;
    pieces += more;
  }
  a.first_piece[a.tensors] = (int)pieces;
  return i;
}
// The workgroups' sums of all tensors; `count` of them.
static int launch_squares(hipStream_t st, int const *dtypes, void const *const *grads, int64_t const *elems, int num, double *partial, int &count) {
  NormTable a;
  count = 0;
  int64_t bytes = 0;
  for (int i = 0; i < num; i++) bytes += elems[i] * (int64_t)dtype_size(dtypes[i]);
  for (int first = 0; first < num;) {
    first = fill_table(a, dtypes, grads, nullptr, elems, num, first, kNormLoads, INT32_MAX);  // (a whole table has fewer)
    int const pieces = a.first_piece[a.tensors], grid = pieces < kNormWorkgroups ? pieces : kNormWorkgroups;
    if (grid == 0) continue;
    if (bytes <= kNormKept) square_sum_kernel<false><<<dim3((unsigned)grid), kNormThreads, 0, st>>>(a, partial + count);
    else square_sum_kernel<true><<<dim3((unsigned)grid), kNormThreads, 0, st>>>(a, partial + count);
    FFK_CHECK_LAUNCH();
    count += grid;
  }
  return FFK_OK;
}

static int check_workspace(char const *who, void const *workspace, size_t bytes, int num) {
  size_t const need = ffk_grad_norm_workspace_bytes(num);
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 8 != 0 || bytes < need) {
    return fail(FFK_ERR_WORKSPACE, "%s: workspace must hold %zu bytes, 8-byte aligned (%zu given)", who, need, workspace == nullptr ? (size_t)0 : bytes);
  }
  return FFK_OK;
}

}  // namespace ffk

using namespace ffk;

extern "C" size_t ffk_grad_norm_workspace_bytes(int num_tensors) {
  // every launch of the norm has a whole table but the last (its pieces are taken in turn, whatever their number)
  static_assert(kNormTensors * kClipPieces * kClipLoads / kNormLoads < INT32_MAX, "pieces of a table");
  int64_t const n = num_tensors > 0 ? num_tensors : 1;
  return (size_t)ceil_div(n, kNormTensors) * kNormWorkgroups * sizeof(double);
}

extern "C" int ffk_global_grad_norm(ffk_stream_t stream, int const *dtypes, void const *const *grads, int64_t const *elems, int num_tensors,
                                    float *norm, void *workspace, size_t workspace_bytes) {
  int rc = check_list("global_grad_norm", dtypes, grads, elems, num_tensors);
  if (rc != FFK_OK) return rc;
  FFK_REQUIRE(norm != nullptr, "global_grad_norm: NULL norm");
  rc = check_workspace("global_grad_norm", workspace, workspace_bytes, num_tensors);
  if (rc != FFK_OK) return rc;
  hipStream_t const st = as_stream(stream);
  double *const partial = static_cast<double *>(workspace);
  int count = 0;
  rc = launch_squares(st, dtypes, grads, elems, num_tensors, partial, count);
  if (rc != FFK_OK) return rc;
  norm_kernel<<<dim3(1), kNormThreads, 0, st>>>(partial, count, norm);
  FFK_CHECK_LAUNCH();
  return FFK_OK;
}

extern "C" int ffk_clip_grad_norm(ffk_stream_t stream, int const *dtypes, void const *const *grads, void *const *clipped, int64_t const *elems,
                                  int num_tensors, float max_norm, float *norm, void *workspace, size_t workspace_bytes) {
  int rc = check_list("clip_grad_norm", dtypes, grads, elems, num_tensors);
  if (rc != FFK_OK) return rc;
  rc = check_list("clip_grad_norm", dtypes, const_cast<void const *const *>(clipped), elems, num_tensors);
  if (rc != FFK_OK) return rc;
  FFK_REQUIRE(max_norm >= 0.0f, "clip_grad_norm: max_norm must not be negative");
  rc = check_apart("clip_grad_norm", dtypes, grads, clipped, elems, num_tensors);
  if (rc != FFK_OK) return rc;
  rc = check_workspace("clip_grad_norm", workspace, workspace_bytes, num_tensors);
  if (rc != FFK_OK) return rc;
  hipStream_t const st = as_stream(stream);
  double *const partial = static_cast<double *>(workspace);
  int count = 0;
  rc = launch_squares(st, dtypes, grads, elems, num_tensors, partial, count);
  if (rc != FFK_OK) return rc;
  if (count == 0) {  // nothing to clip
    if (norm != nullptr) {
      norm_kernel<<<dim3(1), kNormThreads, 0, st>>>(partial, 0, norm);
      FFK_CHECK_LAUNCH();
    }
    return FFK_OK;
  }
  NormTable a;
  for (int first = 0; first < num_tensors;) {
    first = fill_table(a, dtypes, grads, clipped, elems, num_tensors, first, kClipLoads, kClipPieces);
    int const pieces = a.first_piece[a.tensors];
    if (pieces == 0) continue;
    clip_kernel<<<dim3((unsigned)pieces), kNormThreads, 0, st>>>(a, partial, count, max_norm, norm);
    FFK_CHECK_LAUNCH();
    norm = nullptr;  // written by the first launch
  }
  return FFK_OK;
}
