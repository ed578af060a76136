// hprms_grad_norm.hip - the norm of a list of gradients and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// The squares are exact in binary64 and are summed there, so neither large nor
// tiny gradients leave the range, whatever their count; the pass is bound by
// HBM (one conversion and one binary64 FMA per element).  The list travels in
// the kernels' argument block (kTensors tensors a launch), so a captured call
// holds its own copy and nothing is uploaded.
//
// The tensors are cut into units of some thousand elements, one workgroup each:
// the hardware starts them in order, so the grid works on one moving stretch of
// memory.  (Workgroups that take units in turn, or a long chunk each, drift
// apart and lose bandwidth: scaling 1.74 GB of bfloat16 into other tensors took
// 643 and 670 us against 596.)  Each workgroup leaves one partial sum; they are
// added in a fixed order, by every workgroup of the scaling kernel itself where
// they are few.
#include <hip/hip_runtime.h>

#include "hprms_device.h"
#include "hprms_host.h"

namespace hprms {
namespace {

typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

constexpr int kTensors = 96;  // per launch: the argument block stays below 4 KiB
constexpr int kBlock = 256;
// Elements a unit.  Small lists: kUnit, for workgroups enough.  Past kLongList
// elements the sum of squares takes kLongUnit (as fast, a quarter of the partial
// sums: 277 + 8 us with the kernel that adds them, against 274 + 17), and so
// does scaling in place, which most steps of a training run end at once, the
// factor being 1: starting and ending the workgroups for 872M elements costs 72
// us at kUnit and 19 at kLongUnit, scaling them 596 and 649.
constexpr int32_t kUnit = 8192;
constexpr int32_t kLongUnit = 32768;
constexpr int64_t kLongList = int64_t(1) << 25;
constexpr int kUnroll = 4;  // 16-byte loads on their way per lane
// Up to this many partial sums each workgroup of the scaling kernel adds them up
// itself (up to 32 KB, from L2); a kernel of their own adds more.
constexpr int64_t kFoldParts = 4096;

struct GradList {
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t count[kTensors];
  int32_t first[kTensors + 1];  // first unit of each tensor, and their number
  uint8_t src_dtype[kTensors], dst_dtype[kTensors];
  int32_t n;
};
static_assert(sizeof(GradList) < 3800, "argument block");

// The tensor that unit b belongs to.
__device__ __forceinline__ int find_tensor(const GradList& l, int b) {
  int lo = 0, hi = l.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= b)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <int DT>
struct Elems {  // 16-bit: 8 elements per 16 bytes
  static constexpr int N = 8;
  typedef uint16_t T;
  __device__ static __forceinline__ void unpack(u32x4 v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Fmt<DT>::lo(v[i]);
      f[2 * i + 1] = Fmt<DT>::hi(v[i]);
    }
  }
  __device__ static __forceinline__ float one(T v) { return Fmt<DT>::one(v); }
  __device__ static __forceinline__ u32x4 pack(const float* f) {
    return u32x4{Fmt<DT>::pack(f[0], f[1]), Fmt<DT>::pack(f[2], f[3]), Fmt<DT>::pack(f[4], f[5]),
                 Fmt<DT>::pack(f[6], f[7])};
  }
  __device__ static __forceinline__ T pack1(float f) { return Fmt<DT>::pack1(f); }
};
template <>
struct Elems<HPRMS_DTYPE_FP32> {
  static constexpr int N = 4;
  typedef float T;
  __device__ static __forceinline__ void unpack(u32x4 v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  }
  __device__ static __forceinline__ float one(T v) { return v; }
  __device__ static __forceinline__ T pack1(float f) { return f; }
};

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (unsigned i = 1; i < blockDim.x / 64; ++i) v += lds[i];
  return v;
}

template <int DT>
__device__ __forceinline__ double squares(u32x4 v) {
  float f[Elems<DT>::N];
  Elems<DT>::unpack(v, f);
  double a = 0.0, b = 0.0;
#pragma unroll
  for (int j = 0; j < Elems<DT>::N; j += 2) {
    a = fma((double)f[j], (double)f[j], a);
    b = fma((double)f[j + 1], (double)f[j + 1], b);
  }
  return a + b;
}

template <int DT>
__device__ __forceinline__ double square_sum(const void* src, int64_t n) {
  using E = Elems<DT>;
  const typename E::T* p = (const typename E::T*)src;
  const int64_t nvec = n / E::N;
  double acc = 0.0;
  int64_t v = threadIdx.x;
  for (; v + (kUnroll - 1) * kBlock < nvec; v += kUnroll * kBlock) {
    u32x4 q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = *(const u32x4_a2*)(p + (v + u * kBlock) * E::N);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) acc += squares<DT>(q[u]);
  }
  for (; v < nvec; v += kBlock) acc += squares<DT>(*(const u32x4_a2*)(p + v * E::N));
  for (int64_t i = nvec * E::N + threadIdx.x; i < n; i += kBlock) {
    const double d = (double)E::one(p[i]);
    acc = fma(d, d, acc);
  }
  return acc;
}

__global__ __launch_bounds__(kBlock) void grad_square_kernel(double* partial, int32_t unit, GradList l) {
  __shared__ double lds[kBlock / 64];
  const int b = blockIdx.x, t = find_tensor(l, b);
  const int64_t at = (int64_t)(b - l.first[t]) * unit;
  const int64_t n = l.count[t] - at < unit ? l.count[t] - at : unit;
  double acc;
  switch (l.src_dtype[t]) {
    case HPRMS_DTYPE_BF16: acc = square_sum<HPRMS_DTYPE_BF16>((const uint16_t*)l.src[t] + at, n); break;
    case HPRMS_DTYPE_FP16: acc = square_sum<HPRMS_DTYPE_FP16>((const uint16_t*)l.src[t] + at, n); break;
    default: acc = square_sum<HPRMS_DTYPE_FP32>((const float*)l.src[t] + at, n); break;
  }
  acc = block_sum(acc, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// The factor as a product of two binary32 numbers: one below binary32's normal
// range, as a norm past 2^126 gives it, would lose its precision in one (x keeps
// it, and y = 2^-64 is exact); otherwise y is 1.
__device__ __forceinline__ float2 factor_of(double total, double max_norm) {
  const double f = max_norm / (total + 1e-6);
  return f > 1.0                    ? float2{1.0f, 1.0f}  // NaN stays
         : f > 0.0 && f < 0x1p-126 ? float2{(float)(f * 0x1p64), 0x1p-64f}
                                   : float2{(float)f, 1.0f};
}

// the sum of all partial sums, on every lane of the workgroup
template <int BLOCK>
__device__ __forceinline__ double sum_parts(const double* partial, int32_t parts, double* lds) {
  constexpr int U = 16;  // loads on their way at once
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += BLOCK * U) {
    double v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = partial[min(i + u * BLOCK, parts - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) acc += i + u * BLOCK < parts ? v[u] : 0.0;
  }
  return block_sum(acc, lds);
}

// The norm from the partial sums and (factor not null) the factor.
__global__ __launch_bounds__(1024) void grad_norm_kernel(const double* partial, int32_t parts, double max_norm,
                                                         float* norm, float2* factor) {
  __shared__ double lds[16];
  const double total = sqrt(sum_parts<1024>(partial, parts, lds));
  if (threadIdx.x != 0) return;
  *norm = (float)total;
  if (factor) *factor = factor_of(total, max_norm);
}

// out = g * factor, one conversion to the output's type
template <int ST, int OT>
__device__ __forceinline__ void scale_unit(const void* src, void* dst, int64_t n, float2 factor) {
  using S = Elems<ST>;
  using O = Elems<OT>;
  const typename S::T* p = (const typename S::T*)src;
  typename O::T* q = (typename O::T*)dst;
  const int64_t nvec = n / S::N;
  auto put = [&](u32x4 in, int64_t v) {
    float f[S::N];
    S::unpack(in, f);
#pragma unroll
    for (int j = 0; j < S::N; ++j) f[j] = f[j] * factor.x * factor.y;
    if constexpr (OT == HPRMS_DTYPE_FP32) {
#pragma unroll
      for (int j = 0; j < S::N; j += 4)
        __builtin_nontemporal_store(u32x4{__float_as_uint(f[j]), __float_as_uint(f[j + 1]), __float_as_uint(f[j + 2]),
                                          __float_as_uint(f[j + 3])},
                                    (u32x4_a2*)(q + v * S::N + j));
    } else {
      __builtin_nontemporal_store(O::pack(f), (u32x4_a2*)(q + v * S::N));
    }
  };
  int64_t v = threadIdx.x;
  for (; v + (kUnroll - 1) * kBlock < nvec; v += kUnroll * kBlock) {
    u32x4 in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) in[u] = *(const u32x4_a2*)(p + (v + u * kBlock) * S::N);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) put(in[u], v + u * kBlock);
  }
  for (; v < nvec; v += kBlock) put(*(const u32x4_a2*)(p + v * S::N), v);
  for (int64_t i = nvec * S::N + threadIdx.x; i < n; i += kBlock) q[i] = O::pack1(S::one(p[i]) * factor.x * factor.y);
}

// FOLD: the factor from the partial sums (and the norm, by workgroup 0 of the
// list's first launch), instead of the one that grad_norm_kernel left.
struct ScaleArgs {
  const float2* factor;
  const double* partial;
  float* norm;  // null: written already
  double max_norm;
  int32_t parts;
  int32_t unit;
};

template <bool FOLD>
__global__ __launch_bounds__(kBlock) void grad_scale_kernel(ScaleArgs a, GradList l) {
  float2 f;
  if constexpr (FOLD) {
    __shared__ double lds[kBlock / 64];
    const double total = sqrt(sum_parts<kBlock>(a.partial, a.parts, lds));
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = (float)total;
    f = factor_of(total, a.max_norm);
  } else {
    f = *a.factor;
  }
  const int b = blockIdx.x, t = find_tensor(l, b);
  if (f.x == 1.0f && l.src[t] == l.dst[t]) return;  // multiplying by 1 in place changes nothing
  const int64_t at = (int64_t)(b - l.first[t]) * a.unit;
  const int64_t n = l.count[t] - at < a.unit ? l.count[t] - at : a.unit;
  const int st = l.src_dtype[t], ot = l.dst_dtype[t];
  const char* src = (const char*)l.src[t] + at * (st == HPRMS_DTYPE_FP32 ? 4 : 2);
  char* dst = (char*)l.dst[t] + at * (ot == HPRMS_DTYPE_FP32 ? 4 : 2);
  if (st == HPRMS_DTYPE_FP32)
    scale_unit<HPRMS_DTYPE_FP32, HPRMS_DTYPE_FP32>(src, dst, n, f);
  else if (st == HPRMS_DTYPE_BF16 && ot == HPRMS_DTYPE_FP32)
    scale_unit<HPRMS_DTYPE_BF16, HPRMS_DTYPE_FP32>(src, dst, n, f);
  else if (st == HPRMS_DTYPE_BF16)
    scale_unit<HPRMS_DTYPE_BF16, HPRMS_DTYPE_BF16>(src, dst, n, f);
  else if (ot == HPRMS_DTYPE_FP32)
    scale_unit<HPRMS_DTYPE_FP16, HPRMS_DTYPE_FP32>(src, dst, n, f);
  else
    scale_unit<HPRMS_DTYPE_FP16, HPRMS_DTYPE_FP16>(src, dst, n, f);
}

// ---- host ------------------------------------------------------------------------------
constexpr int64_t kMaxElements = int64_t(1) << 42;  // units and their numbers stay within 31 bits

int64_t units_of(int64_t count, int64_t unit) { return (count + unit - 1) / unit; }

int check_counts(const int64_t* counts, int n) {
  if (n < 0) return fail(HPRMS_E_INVALID, "the number of tensors must be >= 0 (got %d)", n);
  if (n > 0 && !counts) return fail(HPRMS_E_INVALID, "null counts array");
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0) return fail(HPRMS_E_INVALID, "tensor %d has %lld elements", i, (long long)counts[i]);
    if (counts[i] > kMaxElements || (total += counts[i]) > kMaxElements)
      return fail(HPRMS_E_RANGE, "the tensors hold more than 2^42 elements");
  }
  return HPRMS_OK;
}

// calls launch(list, units, launch number) for every kTensors non-empty tensors
template <class Fn>
int each_list(int64_t unit, void* const* outs, const int* out_dtypes, const void* const* grads, const int* dtypes,
              const int64_t* counts, int n, Fn&& launch) {
  GradList l;
  int number = 0;
  int32_t units = 0;
  l.n = 0;
  for (int i = 0; i <= n; ++i) {
    if (l.n == kTensors || (i == n && l.n > 0)) {
      l.first[l.n] = units;
      const int rc = launch(l, units, number++);
      if (rc != HPRMS_OK) return rc;
      units = 0;
      l.n = 0;
    }
    if (i == n || counts[i] == 0) continue;
    l.src[l.n] = grads ? grads[i] : nullptr;
    l.dst[l.n] = outs ? outs[i] : nullptr;
    l.count[l.n] = counts[i];
    l.src_dtype[l.n] = (uint8_t)(dtypes ? dtypes[i] : 0);
    l.dst_dtype[l.n] = (uint8_t)(outs ? out_dtypes[i] : l.src_dtype[l.n]);
    l.first[l.n] = units;
    units += (int32_t)units_of(counts[i], unit);
    ++l.n;
  }
  return HPRMS_OK;
}

int64_t total_of(const int64_t* counts, int n) {
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += counts[i];
  return total;
}

// (and at most 2^16 partial sums and one per tensor, however long the list)
int32_t square_unit(int64_t total) {
  if (total <= kLongList) return kUnit;
  const int64_t unit = ((total >> 16) + kUnit - 1) / kUnit * kUnit;
  return unit > kLongUnit ? (int32_t)unit : kLongUnit;
}

// partial sums over all launches
int64_t parts_of(const int64_t* counts, int n) {
  const int32_t unit = square_unit(total_of(counts, n));
  int64_t parts = 0;
  for (int i = 0; i < n; ++i) parts += units_of(counts[i], unit);
  return parts;
}

// the two leading slots hold the factor
int64_t grad_workspace(int64_t parts) { return 16 + parts * 8; }

bool is_grad_dtype(int d) { return d == HPRMS_DTYPE_BF16 || d == HPRMS_DTYPE_FP16 || d == HPRMS_DTYPE_FP32; }

int run_norm(float* norm, void* const* outs, const int* out_dtypes, const void* const* grads, const int* dtypes,
             const int64_t* counts, int n, double max_norm, void* workspace, int64_t workspace_size,
             hipStream_t stream) {
  int rc = check_counts(counts, n);
  if (rc != HPRMS_OK) return rc;
  if (n > 0 && (!grads || !dtypes)) return fail(HPRMS_E_INVALID, "null tensor array");
  for (int i = 0; i < n; ++i) {
    if (!is_grad_dtype(dtypes[i]))
      return fail(HPRMS_E_INVALID, "tensor %d: dtype must be HPRMS_DTYPE_BF16, _FP16 or _FP32 (got %d)", i, dtypes[i]);
    if (outs && out_dtypes[i] != dtypes[i] && out_dtypes[i] != HPRMS_DTYPE_FP32)
      return fail(HPRMS_E_INVALID, "output %d: dtype must be the gradient's or HPRMS_DTYPE_FP32 (got %d)", i,
                  out_dtypes[i]);
    if (counts[i] == 0) continue;
    if (!grads[i] || (outs && !outs[i])) return fail(HPRMS_E_INVALID, "null tensor pointer (tensor %d)", i);
    if (outs && outs[i] == grads[i] && out_dtypes[i] != dtypes[i])
      return fail(HPRMS_E_INVALID, "output %d lies on its gradient but has another dtype", i);
    if (((uintptr_t)grads[i] & (dtypes[i] == HPRMS_DTYPE_FP32 ? 3 : 1)) != 0 ||
        (outs && ((uintptr_t)outs[i] & (out_dtypes[i] == HPRMS_DTYPE_FP32 ? 3 : 1)) != 0))
      return fail(HPRMS_E_INVALID, "tensor %d is not aligned to its elements", i);
  }
  if (!norm || ((uintptr_t)norm & 3) != 0) return fail(HPRMS_E_INVALID, "norm must point to a float32");
  const int64_t parts = parts_of(counts, n), need = grad_workspace(parts);
  if (!workspace || workspace_size < need || ((uintptr_t)workspace & 15) != 0)
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 16-byte aligned (got %lld)", (long long)need,
                (long long)workspace_size);
  float2* factor = outs ? (float2*)workspace : nullptr;
  double* partial = (double*)((char*)workspace + 16);
  int64_t done = 0;
  const int64_t total = total_of(counts, n);
  const int32_t unit = square_unit(total);
  rc = each_list(unit, outs, out_dtypes, grads, dtypes, counts, n, [&](const GradList& l, int32_t units, int) {
    grad_square_kernel<<<dim3((unsigned)units), dim3(kBlock), 0, stream>>>(partial + done, unit, l);
    done += units;
    return check_launch("gradient norm kernel");
  });
  if (rc != HPRMS_OK) return rc;
  const bool fold = outs && parts > 0 && parts <= kFoldParts;
  if (!fold) {
    grad_norm_kernel<<<dim3(1), dim3(1024), 0, stream>>>(partial, (int32_t)parts, max_norm, norm, factor);
    rc = check_launch("gradient norm kernel");
  }
  if (rc != HPRMS_OK || !outs) return rc;
  bool in_place = true;
  for (int i = 0; i < n; ++i) in_place = in_place && (counts[i] == 0 || outs[i] == grads[i]);
  const int32_t scale_unit = in_place && total > kLongList ? kLongUnit : kUnit;
  return each_list(scale_unit, outs, out_dtypes, grads, dtypes, counts, n,
                   [&](const GradList& l, int32_t units, int number) {
    const ScaleArgs a{factor, partial, number == 0 ? norm : nullptr, max_norm, (int32_t)parts, scale_unit};
    const dim3 groups((unsigned)units);
    if (fold)
      grad_scale_kernel<true><<<groups, dim3(kBlock), 0, stream>>>(a, l);
    else
      grad_scale_kernel<false><<<groups, dim3(kBlock), 0, stream>>>(a, l);
    return check_launch("gradient clipping kernel");
  });
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_grad_norm_workspace(const int64_t* counts, int n) {
  const int rc = check_counts(counts, n);
  return rc != HPRMS_OK ? rc : grad_workspace(parts_of(counts, n));
}

int hprms_grad_norm(float* norm, const void* const* grads, const int* dtypes, const int64_t* counts, int n,
                    void* workspace, int64_t workspace_size, hipStream_t stream) {
  return run_norm(norm, nullptr, nullptr, grads, dtypes, counts, n, 0.0, workspace, workspace_size, stream);
}

int hprms_clip_grad_norm(float* norm, void* const* outs, const int* out_dtypes, const void* const* grads,
                         const int* dtypes, const int64_t* counts, int n, double max_norm, void* workspace,
                         int64_t workspace_size, hipStream_t stream) {
  if (!(max_norm >= 0.0)) return fail(HPRMS_E_INVALID, "max_norm must be >= 0");
  if (n > 0 && (!outs || !out_dtypes)) return fail(HPRMS_E_INVALID, "null output array");
  static void* const none[1] = {nullptr};
  static const int none_dtype[1] = {0};
  return run_norm(norm, n > 0 ? outs : none, n > 0 ? out_dtypes : none_dtype, grads, dtypes, counts, n, max_norm,
                  workspace, workspace_size, stream);
}

}  // extern "C"
