// hprms_norm_add.hip - the edge between two blocks: the norm behind a block, its
// gate, the scaled residual and the norm before the next block, with a 16-bit or
// an 8-bit integer output.
//
// With x the block's output, s the residual, g the gate, a the residual's scale
// and i(v) = 1 / sqrt(mean(v^2) + eps):
//
//   n = x * i(x) * post_weight   (n = x without post_weight)
//   h = rne(a * s + g * n)       the updated residual
//   y = rne(h * i(h) * weight)
//
// and for the integer output, from the 16-bit y as the FP8 forms have it,
// scale = max(max|y| / 127, FLT_MIN) per row and q = rne(clamp(y * (1 / scale))).
//
// x and s are read once and held in registers over the two sums (and the row
// maximum); h and y are written once: 4 rows of traffic a row (3.5 with 8-bit
// output, 5 with a gate for each element), which HBM bounds.  The weights and a
// gate that rows share come from L2.
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_rows.h"

namespace hprms {
namespace {

struct NormAddArgs {
  const uint16_t* input;
  const uint16_t* residual;
  void* out;  // 16-bit, or int8 elements
  uint16_t* residual_out;
  const uint16_t* weight;
  const uint16_t* post_weight;  // null: no norm behind the block
  const uint16_t* gate;         // null: none
  float* scale;                 // int8 output
  int64_t rows, rows_per_gate;  // row r has the gate's row r / rows_per_gate
  int64_t row_from;             // the launch's first row
  int64_t input_stride, residual_stride, out_stride, residual_out_stride, gate_stride;
  int32_t hidden;
  float eps, residual_scale;
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int64_t gate_row(const NormAddArgs& a, int64_t row) {
  // one gate for all rows, or one for each, or one for every so many
  if (a.rows_per_gate >= a.rows) return 0;
  if (a.rows_per_gate == 1) return row;
  return (a.rows | a.rows_per_gate) >> 31 ? row / a.rows_per_gate : (int64_t)((uint32_t)row / (uint32_t)a.rows_per_gate);
}

__device__ __forceinline__ float inverse_rms(float squares, int32_t hidden, float eps) {
  return 1.0f / sqrtf(squares / (float)hidden + eps);
}

// A row's scale and its reciprocal from the 16 bits of max |y|; a row that holds NaN
// or infinity has that as its scale, and zeros as elements.
struct RowScale {
  float scale, inverse;
  bool finite;
};
template <int DT>
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float amax = Fmt<DT>::lo(top);
  const bool finite = __float_as_uint(amax) < 0x7f800000u;
  const float scale = finite ? fmaxf(amax / 127.0f, 1.17549435e-38f) : amax;
  return {scale, finite ? 1.0f / scale : 0.0f, finite};
}

// v in [-127.5, 127.5] to the nearest integer, ties to even, in the low byte: 1.5 *
// 2^23 leaves no fraction bits.
__device__ __forceinline__ uint32_t to_int8(float v, const RowScale& s) {
  const float c = __builtin_amdgcn_fmed3f(v * s.inverse, -127.0f, 127.0f);
  return s.finite ? __float_as_uint(c + 12582912.0f) & 0xffu : 0u;
}

template <int DT, int LPR, int VPL, int BLOCK, bool POST, bool INT8, bool NT>
__global__ __launch_bounds__(BLOCK) void norm_add_kernel(NormAddArgs a) {
  constexpr int RPB = BLOCK / LPR;
  __shared__ float sums[2][BLOCK / 64];
  __shared__ uint32_t tops[BLOCK / 64];
  const int lane = threadIdx.x % LPR;
  const int64_t row = a.row_from + (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const bool live = RPB == 1 || row < a.rows;
  const int nvec = a.hidden >> 3, tail = a.hidden & 7;
  const int dup = tail ? 8 - tail : 0;  // the tail vector's elements that a whole vector holds
  const uint16_t* gate = a.gate ? a.gate + gate_row(a, live ? row : 0) * a.gate_stride : nullptr;
  int off[VPL], skip[VPL];
  bool on[VPL];
  u32x4 x[VPL], s[VPL];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int v = k * LPR + lane;
    on[k] = live && v < nvec + (tail ? 1 : 0);
    off[k] = v < nvec ? v * 8 : a.hidden - 8;
    skip[k] = v < nvec ? 0 : dup;
    x[k] = s[k] = u32x4{0, 0, 0, 0};
    if (on[k]) {
      x[k] = load_row8_once<NT>(a.input + row * a.input_stride + off[k]);
      s[k] = load_row8_once<NT>(a.residual + row * a.residual_stride + off[k]);
    }
    if (tail) {
      drop_first(x[k], skip[k]);
      drop_first(s[k], skip[k]);
    }
  }
  float ix = 1.0f;
  if constexpr (POST) {
    float ss[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = element<DT>(x[k], j);
        ss[0] += v * v;
      }
    sum_rows<1, LPR, BLOCK>(ss, sums[0]);
    ix = inverse_rms(ss[0], a.hidden, a.eps);
  }
  float ss[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    u32x4 p = {0, 0, 0, 0}, g = {0, 0, 0, 0};
    packed_again(x[k]);
    packed_again(s[k]);
    if (POST && on[k]) p = load_row8(a.post_weight + off[k]);
    if (gate && on[k]) g = load_row8(gate + off[k]);
    float h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float n = element<DT>(x[k], j);
      if constexpr (POST) n = n * ix * element<DT>(p, j);
      if (gate) n *= element<DT>(g, j);
      h[j] = element<DT>(s[k], j) * a.residual_scale + n;
    }
    s[k] = pack8<DT>(h);
    if (skip[k] > 0) drop_first(s[k], skip[k]);  // (0 times an infinite gate or weight: NaN)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = element<DT>(s[k], j);
      ss[0] += v * v;
    }
    if (on[k]) store_row8(a.residual_out + row * a.residual_out_stride + off[k], s[k], skip[k]);
  }
  u32x4 w[VPL];
#pragma unroll
  for (int k = 0; k < VPL; ++k) w[k] = on[k] ? load_row8(a.weight + off[k]) : u32x4{0, 0, 0, 0};
  sum_rows<1, LPR, BLOCK>(ss, sums[1]);
  const float ih = inverse_rms(ss[0], a.hidden, a.eps);
  u16x2 top = {0, 0};
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = element<DT>(s[k], j) * ih * element<DT>(w[k], j);
    s[k] = pack8<DT>(y);
    if constexpr (INT8) {
      if (skip[k] > 0) drop_first(s[k], skip[k]);  // (0 times an infinite weight or ih)
      u16x2 t = {0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, s[k][j] & 0x7fff7fffu));
      top = on[k] ? __builtin_elementwise_max(top, t) : top;
    } else if (on[k]) {
      store_row8((uint16_t*)a.out + row * a.out_stride + off[k], s[k], skip[k]);
    }
  }
  if constexpr (INT8) {
    const RowScale q =
        row_scale<DT>(max_rows<LPR, BLOCK>(__builtin_elementwise_max((uint32_t)top[0], (uint32_t)top[1]), tops));
    if (live && lane == 0) a.scale[row] = q.scale;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      if (!on[k]) continue;
      u32x2 b = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j / 4] |= to_int8(element<DT>(s[k], j), q) << (8 * (j & 3));
      int8_t* to = (int8_t*)a.out + row * a.out_stride + off[k];
      if (skip[k] == 0) {
        __builtin_nontemporal_store(b, (u32x2_any*)to);
      } else {
#pragma unroll
        for (int j = 1; j < 8; ++j)
          if (j >= skip[k]) to[j] = (int8_t)(b[j / 4] >> (8 * (j & 3)));
      }
    }
  }
}

// ---- any width: passes over the row ----------------------------------------------------
// Rows of fewer than 8 or more than 32768 elements, one workgroup each.  A lane
// reads and writes the same elements in every pass.
template <int DT, bool POST, bool INT8>
__global__ __launch_bounds__(256) void norm_add_any_kernel(NormAddArgs a) {
  using F = Fmt<DT>;
  __shared__ float sums[2][4];
  __shared__ uint32_t tops[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint16_t* x = a.input + row * a.input_stride;
    const uint16_t* s = a.residual + row * a.residual_stride;
    const uint16_t* gate = a.gate ? a.gate + gate_row(a, row) * a.gate_stride : nullptr;
    uint16_t* h = a.residual_out + row * a.residual_out_stride;
    __syncthreads();  // the row before has read the sums
    float ix = 1.0f;
    if constexpr (POST) {
      float ss[1] = {0.0f};
      for (int32_t i = threadIdx.x; i < a.hidden; i += 256) ss[0] += F::one(x[i]) * F::one(x[i]);
      sum_rows<1, 256, 256>(ss, sums[0]);
      ix = inverse_rms(ss[0], a.hidden, a.eps);
    }
    float ss[1] = {0.0f};
    for (int32_t i = threadIdx.x; i < a.hidden; i += 256) {
      float n = F::one(x[i]);
      if constexpr (POST) n = n * ix * F::one(a.post_weight[i]);
      if (gate) n *= F::one(gate[i]);
      const uint16_t v = F::pack1(F::one(s[i]) * a.residual_scale + n);
      h[i] = v;
      ss[0] += F::one(v) * F::one(v);
    }
    sum_rows<1, 256, 256>(ss, sums[1]);
    const float ih = inverse_rms(ss[0], a.hidden, a.eps);
    if constexpr (!INT8) {
      uint16_t* out = (uint16_t*)a.out + row * a.out_stride;
      for (int32_t i = threadIdx.x; i < a.hidden; i += 256)
        out[i] = F::pack1(F::one(h[i]) * ih * F::one(a.weight[i]));
    } else {
      int8_t* out = (int8_t*)a.out + row * a.out_stride;
      uint32_t top = 0;
      for (int32_t i = threadIdx.x; i < a.hidden; i += 256)
        top = __builtin_elementwise_max(top, (uint32_t)F::pack1(F::one(h[i]) * ih * F::one(a.weight[i])) & 0x7fffu);
      const RowScale q = row_scale<DT>(max_rows<256, 256>(top, tops));
      if (threadIdx.x == 0) a.scale[row] = q.scale;
      for (int32_t i = threadIdx.x; i < a.hidden; i += 256)
        out[i] = (int8_t)to_int8(F::one(F::pack1(F::one(h[i]) * ih * F::one(a.weight[i]))), q);
    }
  }
}

// ---- host ------------------------------------------------------------------------------
constexpr int64_t kMaxHidden = int64_t(1) << 24;
constexpr int64_t kVectorHidden = 32768;

// a launch holds fewer than 2^32 work-items
constexpr int64_t kMaxGroups = int64_t(1) << 21;

template <int DT, bool POST, bool INT8, int LPR, int VPL, int BLOCK>
void launch(NormAddArgs a, hipStream_t stream) {
  constexpr int RPB = BLOCK / LPR;
  const int64_t groups = (a.rows + RPB - 1) / RPB;
  const bool nt = past_caches(a.rows, a.hidden, {{a.input, a.input_stride}, {a.residual, a.residual_stride}});
  for (int64_t from = 0; from < groups; from += kMaxGroups) {
    const dim3 grid((unsigned)(groups - from < kMaxGroups ? groups - from : kMaxGroups)), block(BLOCK);
    a.row_from = from * RPB;
    if (nt)
      norm_add_kernel<DT, LPR, VPL, BLOCK, POST, INT8, true><<<grid, block, 0, stream>>>(a);
    else
      norm_add_kernel<DT, LPR, VPL, BLOCK, POST, INT8, false><<<grid, block, 0, stream>>>(a);
  }
}

// Shapes go by the width alone, so a row's bits do not depend on the call's rows;
// each is the fastest of those tried, or within 3% of it.  Lanes a row x vectors a
// lane, bf16 with both norms, 33.5M elements (268 MB) or as many rows as noted, us:
//   128 16 x 1 44.6; 256 32 x 1 44.4; 512 64 x 1 44.7; 1024 64 x 2 44.8
//   2048 128 x 2 44.9; 4096 256 x 2 45.9, 512 x 1 45.2, 128 x 4 48.3, but with 8-bit
//   output 256 x 2 42.0, 512 x 1 46.4
//   5120 (5000 rows) 256 x 3 36.4, 384 x 2 37.6, 512 x 2 38.8; 6144 256 x 3 43.0
//   8192 512 x 2 46.5, 256 x 4 46.7, 1024 x 1 48.6
//   12288 512 x 4 49.0, 512 x 3 47.5; 16384 512 x 4 48.3, 1024 x 2 47.9; 32768 1024 x 4 49.8
template <int DT, bool POST, bool INT8>
int launch_all(const NormAddArgs& a, hipStream_t stream) {
  const int32_t slots = (a.hidden + 7) / 8;
  if (a.hidden < 8 || a.hidden > kVectorHidden)
    norm_add_any_kernel<DT, POST, INT8><<<dim3((unsigned)(a.rows < 8192 ? a.rows : 8192)), dim3(256), 0, stream>>>(a);
  else if (slots <= 16)
    launch<DT, POST, INT8, 16, 1, 256>(a, stream);
  else if (slots <= 32)
    launch<DT, POST, INT8, 32, 1, 256>(a, stream);
  else if (slots <= 64)
    launch<DT, POST, INT8, 64, 1, 256>(a, stream);
  else if (slots <= 128)
    launch<DT, POST, INT8, 64, 2, 256>(a, stream);
  else if (slots <= 256)
    launch<DT, POST, INT8, 128, 2, 128>(a, stream);
  else if (slots <= 512)
    launch<DT, POST, INT8, 256, 2, 256>(a, stream);
  else if (slots <= 768)
    launch<DT, POST, INT8, 256, 3, 256>(a, stream);
  else if (slots <= 1024)
    launch<DT, POST, INT8, 512, 2, 512>(a, stream);
  else if (slots <= 2048)
    launch<DT, POST, INT8, 512, 4, 512>(a, stream);
  else
    launch<DT, POST, INT8, 1024, 4, 1024>(a, stream);
  return check_launch("norm + gate + add + norm kernel");
}

template <int DT>
int launch_kind(const NormAddArgs& a, hipStream_t stream) {
  if (a.scale) return a.post_weight ? launch_all<DT, true, true>(a, stream) : launch_all<DT, false, true>(a, stream);
  return a.post_weight ? launch_all<DT, true, false>(a, stream) : launch_all<DT, false, false>(a, stream);
}

int check(const NormAddArgs& a, int64_t hidden, int dtype, bool int8, double eps, double residual_scale) {
  if (dtype != HPRMS_DTYPE_BF16 && dtype != HPRMS_DTYPE_FP16)
    return fail(HPRMS_E_INVALID, "dtype must be HPRMS_DTYPE_BF16 or HPRMS_DTYPE_FP16 (got %d)", dtype);
  if (a.rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)a.rows);
  if (hidden < 1) return fail(HPRMS_E_INVALID, "hidden must be >= 1 (got %lld)", (long long)hidden);
  if (hidden > kMaxHidden)
    return fail(HPRMS_E_RANGE, "hidden %lld exceeds the supported maximum %lld", (long long)hidden,
                (long long)kMaxHidden);
  if (a.rows >= int64_t(1) << 31) return fail(HPRMS_E_RANGE, "rows %lld exceed 2^31 - 1", (long long)a.rows);
  if (a.input_stride < hidden || a.residual_stride < hidden || a.out_stride < hidden ||
      a.residual_out_stride < hidden || (a.gate && a.gate_stride < hidden))
    return fail(HPRMS_E_INVALID, "row strides must be >= hidden");
  if (a.gate && a.rows_per_gate < 1)
    return fail(HPRMS_E_INVALID, "rows_per_gate must be >= 1 (got %lld)", (long long)a.rows_per_gate);
  if (!(eps >= 0.0)) return fail(HPRMS_E_INVALID, "eps must be >= 0");
  if (!(residual_scale - residual_scale == 0.0)) return fail(HPRMS_E_INVALID, "residual_scale must be finite");
  for (int64_t stride : {a.input_stride, a.residual_stride, a.out_stride, a.residual_out_stride})
    if (!extent_ok(a.rows, stride, 2, hidden))
      return fail(HPRMS_E_RANGE, "%lld rows at these row strides span more than 2^56 bytes", (long long)a.rows);
  if (a.gate && a.rows > 0 && !extent_ok((a.rows - 1) / a.rows_per_gate + 1, a.gate_stride, 2, hidden))
    return fail(HPRMS_E_RANGE, "the gate's rows at their stride span more than 2^56 bytes");
  if (a.rows == 0) return HPRMS_OK;
  if (!a.input || !a.residual || !a.out || !a.residual_out || !a.weight || (int8 && !a.scale))
    return fail(HPRMS_E_INVALID, "null tensor pointer");
  if ((((uintptr_t)a.input | (uintptr_t)a.residual | (uintptr_t)a.residual_out | (uintptr_t)a.weight |
        (uintptr_t)a.post_weight | (uintptr_t)a.gate) & 1) != 0 || (!int8 && ((uintptr_t)a.out & 1) != 0) ||
      ((uintptr_t)a.scale & 3) != 0)
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  if (a.out == a.residual_out || a.out == a.residual || a.residual_out == a.input || (int8 && a.out == a.input))
    return fail(HPRMS_E_INVALID, "outputs alias each other or another row tensor than their own");
  if (a.rows > 1 && ((a.out == a.input && a.out_stride != a.input_stride) ||
                     (a.residual_out == a.residual && a.residual_out_stride != a.residual_stride)))
    return fail(HPRMS_E_INVALID, "an in-place alias needs equal row strides");
  return HPRMS_OK;
}

}  // namespace
}  // namespace hprms

using namespace hprms;

namespace {

int run(void* out, float* scale, bool int8, void* residual_out, const void* input, const void* post_weight,
        const void* weight, const void* residual, const void* gate, int64_t rows, int64_t hidden, int64_t rows_per_gate,
        int64_t out_row_stride, int64_t residual_out_row_stride, int64_t input_row_stride,
        int64_t residual_row_stride, int64_t gate_row_stride, int dtype, double residual_scale, double eps,
        hipStream_t stream) {
  NormAddArgs a = {};
  a.input = (const uint16_t*)input;
  a.residual = (const uint16_t*)residual;
  a.out = out;
  a.residual_out = (uint16_t*)residual_out;
  a.weight = (const uint16_t*)weight;
  a.post_weight = (const uint16_t*)post_weight;
  a.gate = (const uint16_t*)gate;
  a.scale = scale;
  a.rows = rows;
  a.rows_per_gate = gate ? rows_per_gate : 1;
  a.input_stride = input_row_stride;
  a.residual_stride = residual_row_stride;
  a.out_stride = out_row_stride;
  a.residual_out_stride = residual_out_row_stride;
  a.gate_stride = gate_row_stride;
  const int rc = check(a, hidden, dtype, int8, eps, residual_scale);
  if (rc != HPRMS_OK || rows == 0) return rc;
  a.hidden = (int32_t)hidden;
  a.eps = (float)eps;
  a.residual_scale = (float)residual_scale;
  return dtype == HPRMS_DTYPE_BF16 ? launch_kind<HPRMS_DTYPE_BF16>(a, stream) : launch_kind<HPRMS_DTYPE_FP16>(a, stream);
}

}  // namespace

extern "C" {

int hprms_norm_add_rmsnorm(void* out, void* residual_out, const void* input, const void* post_weight,
                           const void* weight, const void* residual, const void* gate, int64_t rows, int64_t hidden,
                           int64_t rows_per_gate, int64_t out_row_stride, int64_t residual_out_row_stride,
                           int64_t input_row_stride, int64_t residual_row_stride, int64_t gate_row_stride, int dtype,
                           double residual_scale, double eps, hipStream_t stream) {
  return run(out, nullptr, false, residual_out, input, post_weight, weight, residual, gate, rows, hidden,
             rows_per_gate, out_row_stride, residual_out_row_stride, input_row_stride, residual_row_stride,
             gate_row_stride, dtype, residual_scale, eps, stream);
}

int hprms_norm_add_rmsnorm_int8(void* out, float* scale, void* residual_out, const void* input,
                                const void* post_weight, const void* weight, const void* residual, const void* gate,
                                int64_t rows, int64_t hidden, int64_t rows_per_gate, int64_t out_row_stride,
                                int64_t residual_out_row_stride, int64_t input_row_stride,
                                int64_t residual_row_stride, int64_t gate_row_stride, int dtype,
                                double residual_scale, double eps, hipStream_t stream) {
  return run(out, scale, true, residual_out, input, post_weight, weight, residual, gate, rows, hidden, rows_per_gate,
             out_row_stride, residual_out_row_stride, input_row_stride, residual_row_stride, gate_row_stride, dtype,
             residual_scale, eps, stream);
}

}  // extern "C"
