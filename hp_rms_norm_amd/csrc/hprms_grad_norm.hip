// hprms_grad_norm.hip - the norm of a list of gradients and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// The squares are exact in binary64 and are summed there, so neither large nor
// tiny gradients leave the range, whatever their count; the pass is bound by
// HBM (one conversion and one binary64 FMA per element).  The list travels in
// the kernels' argument block (kTensors tensors a launch), so a captured call
// holds its own copy and nothing is uploaded.  Each workgroup takes one chunk
// of one tensor and writes one partial sum; a one-workgroup kernel adds them
// in a fixed order.
#include <hip/hip_runtime.h>

#include "hprms_device.h"
#include "hprms_host.h"

namespace hprms {
namespace {

typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

constexpr int kTensors = 96;  // per launch: the argument block stays below 4 KiB
constexpr int kBlock = 256;
constexpr int64_t kMinChunk = 8192;     // elements per workgroup, at least
constexpr int64_t kMaxChunks = 1 << 14;  // workgroups over the whole list, about

struct GradList {
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t count[kTensors];
  int32_t first[kTensors + 1];  // first workgroup of each tensor
  uint8_t src_dtype[kTensors], dst_dtype[kTensors];
  int32_t n;
};
static_assert(sizeof(GradList) < 3800, "argument block");

// The tensor whose chunks hold workgroup b.
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
__device__ __forceinline__ double square_sum(const void* src, int64_t n) {
  using E = Elems<DT>;
  const typename E::T* p = (const typename E::T*)src;
  const int64_t nvec = n / E::N;
  double acc = 0.0;
  for (int64_t v = threadIdx.x; v < nvec; v += kBlock) {
    float f[E::N];
    E::unpack(*(const u32x4_a2*)(p + v * E::N), f);
#pragma unroll
    for (int j = 0; j < E::N; ++j) acc = fma((double)f[j], (double)f[j], acc);
  }
  for (int64_t i = nvec * E::N + threadIdx.x; i < n; i += kBlock) {
    const double d = (double)E::one(p[i]);
    acc = fma(d, d, acc);
  }
  return acc;
}

__global__ __launch_bounds__(kBlock) void grad_square_kernel(double* partial, int64_t chunk, GradList l) {
  __shared__ double lds[kBlock / 64];
  const int b = blockIdx.x;
  const int t = find_tensor(l, b);
  const int64_t at = (int64_t)(b - l.first[t]) * chunk;
  const int64_t n = l.count[t] - at < chunk ? l.count[t] - at : chunk;
  double acc;
  switch (l.src_dtype[t]) {
    case HPRMS_DTYPE_BF16: acc = square_sum<HPRMS_DTYPE_BF16>((const uint16_t*)l.src[t] + at, n); break;
    case HPRMS_DTYPE_FP16: acc = square_sum<HPRMS_DTYPE_FP16>((const uint16_t*)l.src[t] + at, n); break;
    default: acc = square_sum<HPRMS_DTYPE_FP32>((const float*)l.src[t] + at, n); break;
  }
  acc = block_sum(acc, lds);
  if (threadIdx.x == 0) partial[b] = acc;
}

// The norm from the partial sums and (factor not null) the factor, as a product
// of two binary32 numbers: a factor below binary32's normal range, as a norm
// past 2^126 gives it, would lose its precision in one (factor.x keeps it, and
// factor.y = 2^-64 is exact); otherwise factor.y is 1.
__global__ __launch_bounds__(1024) void grad_norm_kernel(const double* partial, int32_t parts, double max_norm,
                                                         float* norm, float2* factor) {
  __shared__ double lds[16];
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += 1024) acc += partial[i];
  acc = block_sum(acc, lds);
  if (threadIdx.x == 0) {
    const double total = sqrt(acc);
    *norm = (float)total;
    if (factor) {
      const double f = max_norm / (total + 1e-6);
      *factor = f > 1.0 ? float2{1.0f, 1.0f}  // NaN stays
                : f > 0.0 && f < 0x1p-126 ? float2{(float)(f * 0x1p64), 0x1p-64f} : float2{(float)f, 1.0f};
    }
  }
}

// out = g * factor, one conversion to the output's type
template <int ST, int OT>
__device__ __forceinline__ void scale_chunk(const void* src, void* dst, int64_t n, float2 factor) {
  using S = Elems<ST>;
  using O = Elems<OT>;
  const typename S::T* p = (const typename S::T*)src;
  typename O::T* q = (typename O::T*)dst;
  const int64_t nvec = n / S::N;
  for (int64_t v = threadIdx.x; v < nvec; v += kBlock) {
    float f[S::N];
    S::unpack(*(const u32x4_a2*)(p + v * S::N), f);
#pragma unroll
    for (int j = 0; j < S::N; ++j) f[j] = f[j] * factor.x * factor.y;
    if constexpr (OT == HPRMS_DTYPE_FP32) {
#pragma unroll
      for (int j = 0; j < S::N; j += 4)
        *(u32x4_a2*)(q + v * S::N + j) = u32x4{__float_as_uint(f[j]), __float_as_uint(f[j + 1]),
                                             __float_as_uint(f[j + 2]), __float_as_uint(f[j + 3])};
    } else {
      *(u32x4_a2*)(q + v * S::N) = O::pack(f);
    }
  }
  for (int64_t i = nvec * S::N + threadIdx.x; i < n; i += kBlock) q[i] = O::pack1(S::one(p[i]) * factor.x * factor.y);
}

__global__ __launch_bounds__(kBlock) void grad_scale_kernel(const float2* factor, int64_t chunk, GradList l) {
  const float2 f = *factor;
  const int b = blockIdx.x;
  const int t = find_tensor(l, b);
  if (f.x == 1.0f && l.src[t] == l.dst[t]) return;  // multiplying by 1 in place changes nothing
  const int64_t at = (int64_t)(b - l.first[t]) * chunk;
  const int64_t n = l.count[t] - at < chunk ? l.count[t] - at : chunk;
  const int st = l.src_dtype[t], ot = l.dst_dtype[t];
  const char* src = (const char*)l.src[t] + at * (st == HPRMS_DTYPE_FP32 ? 4 : 2);
  char* dst = (char*)l.dst[t] + at * (ot == HPRMS_DTYPE_FP32 ? 4 : 2);
  if (st == HPRMS_DTYPE_FP32)
    scale_chunk<HPRMS_DTYPE_FP32, HPRMS_DTYPE_FP32>(src, dst, n, f);
  else if (st == HPRMS_DTYPE_BF16 && ot == HPRMS_DTYPE_FP32)
    scale_chunk<HPRMS_DTYPE_BF16, HPRMS_DTYPE_FP32>(src, dst, n, f);
  else if (st == HPRMS_DTYPE_BF16)
    scale_chunk<HPRMS_DTYPE_BF16, HPRMS_DTYPE_BF16>(src, dst, n, f);
  else if (ot == HPRMS_DTYPE_FP32)
    scale_chunk<HPRMS_DTYPE_FP16, HPRMS_DTYPE_FP32>(src, dst, n, f);
  else
    scale_chunk<HPRMS_DTYPE_FP16, HPRMS_DTYPE_FP16>(src, dst, n, f);
}

// ---- host ------------------------------------------------------------------------------
// Elements per workgroup: the whole list in about kMaxChunks workgroups at most.
int64_t chunk_of(int64_t total) {
  const int64_t c = (total / kMaxChunks + kMinChunk - 1) / kMinChunk * kMinChunk;
  return c < kMinChunk ? kMinChunk : c;
}

struct Plan {
  int64_t total, chunk, parts;
};

int plan_of(const int64_t* counts, int n, Plan* p) {
  if (n < 0) return fail(HPRMS_E_INVALID, "the number of tensors must be >= 0 (got %d)", n);
  if (n > 0 && !counts) return fail(HPRMS_E_INVALID, "null counts array");
  p->total = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0) return fail(HPRMS_E_INVALID, "tensor %d has %lld elements", i, (long long)counts[i]);
    if (counts[i] > (int64_t(1) << 48) || p->total > (int64_t(1) << 48))
      return fail(HPRMS_E_RANGE, "the tensors hold more than 2^48 elements");
    p->total += counts[i];
  }
  p->chunk = chunk_of(p->total);
  p->parts = 0;
  for (int i = 0; i < n; ++i) p->parts += (counts[i] + p->chunk - 1) / p->chunk;
  return HPRMS_OK;
}

// the two leading slots hold the factor
int64_t grad_workspace(const Plan& p) { return 16 + p.parts * 8; }

bool is_grad_dtype(int d) { return d == HPRMS_DTYPE_BF16 || d == HPRMS_DTYPE_FP16 || d == HPRMS_DTYPE_FP32; }

// calls launch(list, workgroups, partials before it) for every kTensors non-empty tensors
template <class Fn>
int each_list(const Plan& p, void* const* outs, const int* out_dtypes, const void* const* grads, const int* dtypes,
              const int64_t* counts, int n, Fn&& launch) {
  GradList l;
  int64_t done = 0;
  int32_t blocks = 0;
  l.n = 0;
  for (int i = 0; i <= n; ++i) {
    if (l.n == kTensors || (i == n && l.n > 0)) {
      l.first[l.n] = blocks;
      const int rc = launch(l, blocks, done);
      if (rc != HPRMS_OK) return rc;
      done += blocks;
      blocks = 0;
      l.n = 0;
    }
    if (i == n || counts[i] == 0) continue;
    l.src[l.n] = grads[i];
    l.dst[l.n] = outs ? outs[i] : nullptr;
    l.count[l.n] = counts[i];
    l.src_dtype[l.n] = (uint8_t)dtypes[i];
    l.dst_dtype[l.n] = (uint8_t)(outs ? out_dtypes[i] : dtypes[i]);
    l.first[l.n] = blocks;
    blocks += (int32_t)((counts[i] + p.chunk - 1) / p.chunk);
    ++l.n;
  }
  return HPRMS_OK;
}

int run_norm(float* norm, void* const* outs, const int* out_dtypes, const void* const* grads, const int* dtypes,
             const int64_t* counts, int n, double max_norm, void* workspace, int64_t workspace_size,
             hipStream_t stream) {
  Plan p;
  int rc = plan_of(counts, n, &p);
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
    if (((uintptr_t)grads[i] & (dtypes[i] == HPRMS_DTYPE_FP32 ? 3 : 1)) != 0 ||
        (outs && ((uintptr_t)outs[i] & (out_dtypes[i] == HPRMS_DTYPE_FP32 ? 3 : 1)) != 0))
      return fail(HPRMS_E_INVALID, "tensor %d is not aligned to its elements", i);
  }
  if (!norm || ((uintptr_t)norm & 3) != 0) return fail(HPRMS_E_INVALID, "norm must point to a float32");
  const int64_t need = grad_workspace(p);
  if (!workspace || workspace_size < need || ((uintptr_t)workspace & 15) != 0)
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 16-byte aligned (got %lld)", (long long)need,
                (long long)workspace_size);
  float2* factor = outs ? (float2*)workspace : nullptr;
  double* partial = (double*)((char*)workspace + 16);
  rc = each_list(p, outs, out_dtypes, grads, dtypes, counts, n, [&](const GradList& l, int32_t blocks, int64_t done) {
    grad_square_kernel<<<dim3((unsigned)blocks), dim3(kBlock), 0, stream>>>(partial + done, p.chunk, l);
    return check_launch("gradient norm kernel");
  });
  if (rc != HPRMS_OK) return rc;
  grad_norm_kernel<<<dim3(1), dim3(1024), 0, stream>>>(partial, (int32_t)p.parts, max_norm, norm, factor);
  rc = check_launch("gradient norm kernel");
  if (rc != HPRMS_OK || !outs) return rc;
  return each_list(p, outs, out_dtypes, grads, dtypes, counts, n, [&](const GradList& l, int32_t blocks, int64_t) {
    grad_scale_kernel<<<dim3((unsigned)blocks), dim3(kBlock), 0, stream>>>(factor, p.chunk, l);
    return check_launch("gradient clipping kernel");
  });
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_grad_norm_workspace(const int64_t* counts, int n) {
  Plan p;
  const int rc = plan_of(counts, n, &p);
  return rc != HPRMS_OK ? rc : grad_workspace(p);
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
