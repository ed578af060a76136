// hprms_norm_grad.hip - the gradient of RMSNorm (plain, and of the fused add +
// RMSNorm, whose input and residual share one gradient).
//
// With s the normalised rows' input (the fused op's updated residual), d the
// gradient of the output, g = d * w, r = 1 / sqrt(mean(s^2) + eps):
//
//   dinput  = r * g - s * (r^3 * sum(g * s) / hidden)  [+ dresidual]
//   dweight = sum over rows of d * s * r
//
// A row's two sums (s^2 and g * s) are reduced together, so each tensor is
// read once and held in registers until the row's gradient is written: 3 or 4
// rows of traffic per row, which HBM bounds.  A workgroup walks rows with a
// fixed stride and keeps its lanes' columns of dweight in binary32 registers;
// it writes them once, at its end, as one row of partial sums, and a second
// kernel adds those rows in a fixed order (no atomics: a call's bits do not
// change from run to run).
#include <hip/hip_runtime.h>

#include "hprms_device.h"
#include "hprms_host.h"

namespace hprms {
namespace {

// 16 bytes at any 2-byte boundary (gfx950 runs global accesses unaligned)
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x4 load_vec(const uint16_t* p) { return *(const u32x4_a2*)p; }
// the row tensors are touched once
template <bool NT>
__device__ __forceinline__ u32x4 load_once(const uint16_t* p) {
  if constexpr (NT)
    return __builtin_nontemporal_load((const u32x4_a2*)p);
  else
    return load_vec(p);
}
__device__ __forceinline__ void store_once(uint16_t* p, u32x4 v) { __builtin_nontemporal_store(v, (u32x4_a2*)p); }

struct NormGradArgs {
  uint16_t* dinput;
  const uint16_t* dout;
  const uint16_t* input;
  const uint16_t* dresidual;  // null: none
  const uint16_t* weight;
  float* partial;             // [gridDim.x, hidden]
  int64_t rows;
  int64_t dinput_stride, dout_stride, input_stride, dresidual_stride;
  int32_t hidden;
  float eps;
};

// Two sums over the LPR lanes of a row at once; every lane gets both.
template <int LPR, int BLOCK>
__device__ __forceinline__ void row_sums(float& a, float& b, float* lds) {
  constexpr int GW = LPR < 64 ? LPR : 64;
  a = group_sum<GW>(a);
  b = group_sum<GW>(b);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    const int wave = threadIdx.x / 64;
    const int row = threadIdx.x / LPR;
    if ((threadIdx.x & 63) == 0) {
      lds[2 * wave] = a;
      lds[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a += lds[2 * (row * W + i)];
      b += lds[2 * (row * W + i) + 1];
    }
  }
}

// LPR lanes per row, VPL vectors of 8 elements per lane: slot v = k * LPR +
// lane holds elements 8v ... 8v + 7; for hidden % 8 != 0 the slot after the
// last whole vector holds the row's last 8 elements, of which only those that
// no whole vector holds count in the sums (the others are stored twice, with
// the same bits).
template <int DT, int LPR, int VPL, int BLOCK, bool AHEAD, bool RES, bool NT>
__global__ __launch_bounds__(BLOCK) void norm_grad_kernel(NormGradArgs a) {
  using F = Fmt<DT>;
  constexpr int RPB = BLOCK / LPR;
  constexpr int SUMS = BLOCK / 64 * 2;
  __shared__ float lds[2][SUMS];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  const int nvec = a.hidden >> 3, tail = a.hidden & 7;
  const int slots = nvec + (tail ? 1 : 0);
  int off[VPL];
  bool on[VPL];
  u32x4 w[VPL];
  // at 4 vectors a lane of 1024 the registers do not hold the sums as well (74-92
  // spilled): they lie in LDS, each lane's own
  constexpr bool LACC = VPL >= 4;
  __shared__ f32x4 lacc[LACC ? VPL * 2 : 1][LACC ? BLOCK : 1];
  float acc[VPL][8];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    if constexpr (LACC) lacc[2 * k][threadIdx.x] = lacc[2 * k + 1][threadIdx.x] = f32x4{0, 0, 0, 0};
    const int v = k * LPR + lane;
    on[k] = v < slots;
    off[k] = v < nvec ? v * 8 : a.hidden - 8;
    w[k] = on[k] ? load_vec(a.weight + off[k]) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.0f;
  }
  // this lane's last slot is the row's tail vector: its first `dup` elements are a whole vector's too
  const int dup = tail ? 8 - tail : 0;
  // the next rows' loads are issued before this row's sums are joined
  u32x4 nx[VPL], nd[VPL], nr[VPL];
  auto load_row = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      nx[k] = nd[k] = nr[k] = u32x4{0, 0, 0, 0};
      if (row < a.rows && on[k]) {
        nx[k] = load_once<NT>(a.input + row * a.input_stride + off[k]);
        nd[k] = load_once<NT>(a.dout + row * a.dout_stride + off[k]);
        if constexpr (RES) nr[k] = load_once<NT>(a.dresidual + row * a.dresidual_stride + off[k]);
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  load_row((int64_t)blockIdx.x * RPB + sub);
  int phase = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + sub;
    const bool live = RPB == 1 || row < a.rows;
    u32x4 x[VPL], d[VPL], r[VPL];
    float ss = 0.0f, gs = 0.0f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      x[k] = nx[k];
      d[k] = nd[k];
      r[k] = nr[k];
    }
    if constexpr (AHEAD) load_row(row + step);
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int skip = tail && k * LPR + lane == nvec ? dup : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xf = j & 1 ? F::hi(x[k][j / 2]) : F::lo(x[k][j / 2]);
        const float df = j & 1 ? F::hi(d[k][j / 2]) : F::lo(d[k][j / 2]);
        const float wf = j & 1 ? F::hi(w[k][j / 2]) : F::lo(w[k][j / 2]);
        if (j >= skip) {
          ss += xf * xf;
          gs += df * wf * xf;
        }
      }
    }
    row_sums<LPR, BLOCK>(ss, gs, lds[phase]);
    phase ^= 1;
    const float rstd = 1.0f / sqrtf(ss / (float)a.hidden + a.eps);
    const float c = rstd * rstd * (rstd * (gs / (float)a.hidden));
    // unpacked again below: the compiler would keep 24 floats a vector over the sums otherwise
#pragma unroll
    for (int k = 0; k < VPL; ++k) asm volatile("" : "+v"(x[k]), "+v"(d[k]), "+v"(w[k]));
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      float o[8], dn[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xf = j & 1 ? F::hi(x[k][j / 2]) : F::lo(x[k][j / 2]);
        const float df = j & 1 ? F::hi(d[k][j / 2]) : F::lo(d[k][j / 2]);
        const float wf = j & 1 ? F::hi(w[k][j / 2]) : F::lo(w[k][j / 2]);
        dn[j] = live ? df * (xf * rstd) : 0.0f;
        o[j] = rstd * (df * wf) - xf * c;
        if constexpr (RES) o[j] += j & 1 ? F::hi(r[k][j / 2]) : F::lo(r[k][j / 2]);
      }
      if constexpr (LACC) {
        lacc[2 * k][threadIdx.x] += f32x4{dn[0], dn[1], dn[2], dn[3]};
        lacc[2 * k + 1][threadIdx.x] += f32x4{dn[4], dn[5], dn[6], dn[7]};
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[k][j] += dn[j];
      }
      if (live && on[k])
        store_once(a.dinput + row * a.dinput_stride + off[k],
                   u32x4{F::pack(o[0], o[1]), F::pack(o[2], o[3]), F::pack(o[4], o[5]), F::pack(o[6], o[7])});
    }
    if constexpr (!AHEAD) load_row(row + step);
  }
  // one row of partial sums per workgroup; the row groups' columns are added through LDS
  __shared__ float cols[RPB > 1 ? RPB * LPR * 8 : 1];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) cols[(sub * LPR + lane) * 8 + j] = acc[k][j];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int i = 1; i < RPB; ++i) acc[k][j] += cols[(i * LPR + lane) * 8 + j];
      }
    }
    if constexpr (LACC) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[k][j] = lacc[2 * k + j / 4][threadIdx.x][j % 4];
    }
    const int skip = tail && k * LPR + lane == nvec ? dup : 0;
    if (sub == 0 && on[k]) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= skip) a.partial[(int64_t)blockIdx.x * a.hidden + off[k] + j] = acc[k][j];
    }
  }
}

// ---- any width: three passes over the rows -----------------------------------------
// Rows of more than 32768 or fewer than 8 elements.  stats[row] = {r, r^3 *
// sum(g * s) / hidden}; the gradient of the weight is summed before dinput is
// written, which may lie on dout.
template <int DT>
__global__ __launch_bounds__(256) void norm_grad_stats_kernel(NormGradArgs a, float2* stats) {
  using F = Fmt<DT>;
  __shared__ float lds[8];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float ss = 0.0f, gs = 0.0f;
    for (int32_t i = threadIdx.x; i < a.hidden; i += 256) {
      const float x = F::one(a.input[row * a.input_stride + i]);
      ss += x * x;
      gs += F::one(a.dout[row * a.dout_stride + i]) * F::one(a.weight[i]) * x;
    }
    __syncthreads();
    row_sums<256, 256>(ss, gs, lds);
    const float rstd = 1.0f / sqrtf(ss / (float)a.hidden + a.eps);
    if (threadIdx.x == 0) stats[row] = float2{rstd, rstd * rstd * (rstd * (gs / (float)a.hidden))};
  }
}

template <int DT>
__global__ __launch_bounds__(256) void norm_grad_columns_kernel(NormGradArgs a, const float2* stats) {
  using F = Fmt<DT>;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.hidden) return;
  float acc = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
    acc += F::one(a.dout[row * a.dout_stride + i]) * (F::one(a.input[row * a.input_stride + i]) * stats[row].x);
  a.partial[(int64_t)blockIdx.y * a.hidden + i] = acc;
}

template <int DT>
__global__ __launch_bounds__(256) void norm_grad_rows_kernel(NormGradArgs a, const float2* stats) {
  using F = Fmt<DT>;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float2 st = stats[row];
    for (int32_t i = threadIdx.x; i < a.hidden; i += 256) {
      float o = st.x * (F::one(a.dout[row * a.dout_stride + i]) * F::one(a.weight[i])) -
                F::one(a.input[row * a.input_stride + i]) * st.y;
      if (a.dresidual) o += F::one(a.dresidual[row * a.dresidual_stride + i]);
      a.dinput[row * a.dinput_stride + i] = F::pack1(o);
    }
  }
}

// ---- dweight from the rows of partial sums -------------------------------------------
// 32 columns per workgroup, 32 lanes' rows apart; the 32 sums of a column are
// added in order.
template <int DT>
__global__ __launch_bounds__(1024) void norm_grad_weight_kernel(const float* partial, int32_t parts, int32_t hidden,
                                                                void* dweight) {
  __shared__ float lds[32][33];
  const int c = threadIdx.x & 31, p = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float acc = 0.0f;
  if (col < hidden) {
    constexpr int U = 8;  // loads on their way at once
    int64_t i = p;
    for (; i + 32 * (U - 1) < parts; i += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = partial[(i + 32 * u) * hidden + col];
#pragma unroll
      for (int u = 0; u < U; ++u) acc += v[u];
    }
    for (; i < parts; i += 32) acc += partial[i * hidden + col];
  }
  lds[p][c] = acc;
  __syncthreads();
  if (p == 0 && col < hidden) {
#pragma unroll
    for (int i = 1; i < 32; ++i) acc += lds[i][c];
    if constexpr (DT == HPRMS_DTYPE_FP32)
      ((float*)dweight)[col] = acc;
    else
      ((uint16_t*)dweight)[col] = Fmt<DT>::pack1(acc);
  }
}

// ---- host ------------------------------------------------------------------------------
constexpr int64_t kMaxGradHidden = int64_t(1) << 24;
constexpr int64_t kVectorHidden = 32768;  // the register-resident kernels' widest rows

// Shapes by width, with the next rows' loads ahead up to 8K.  Few workgroups a
// CU measured best: each adds a row of partial sums, which is written and read
// again.  Times of the row kernel on bf16 rows with dresidual, lanes x vectors
// x workgroup x workgroups per CU (268 MB each): 8192 x 4096 512 x 1 x 512 x 2
// 52.5 us, 256 x 2 x 512 x 1 57.4, 256 x 2 x 256 x 3 56.4; 16384 x 2048 128 x 2
// x 256 x 2 48.9, 128 x 2 x 512 x 1 57.0; 32768 x 1024 64 x 2 x 512 x 1 49.5,
// 64 x 2 x 256 x 4 51.6; 4096 x 8192 512 x 2 x 512 x 1 59.4, two of them 60.3.
// Odd rows of 4097 and rows of 128 are within 2% between their candidates.  From
// 8K the registers do not hold a second row (2048 x 16384: 61.1 us, 62.9 with
// the loads ahead).
struct Shape {
  int lpr, vpl, block, per_cu;
};

Shape shape_of(int64_t hidden) {
  const int64_t slots = (hidden + 7) / 8;
  if (slots <= 16) return {16, 1, 256, 4};
  if (slots <= 32) return {32, 1, 256, 4};
  if (slots <= 64) return {64, 1, 256, 4};
  if (slots <= 128) return {64, 2, 512, 1};
  if (slots <= 256) return {128, 2, 256, 2};
  if (slots <= 512) return {512, 1, 512, 2};
  if (slots <= 768) return {256, 3, 512, 1};
  if (slots <= 1024) return {512, 2, 512, 1};
  if (slots <= 2048) return {1024, 2, 1024, 1};
  return {1024, 4, 1024, 1};
}

bool is_general(int64_t hidden) { return hidden < 8 || hidden > kVectorHidden; }

// workgroups of the row kernel, one row of partial sums each
int64_t grid_of(int64_t rows, int64_t hidden) {
  if (is_general(hidden)) return rows < 64 ? rows : 64;
  const Shape s = shape_of(hidden);
  const int64_t rpb = s.block / s.lpr;
  const int64_t groups = (rows + rpb - 1) / rpb;
  const int64_t most = (int64_t)current_cus() * s.per_cu;
  return groups < most ? groups : most;
}

int64_t workspace_bytes(int64_t rows, int64_t hidden) {
  int64_t n = grid_of(rows, hidden) * hidden * 4;
  if (is_general(hidden)) n += ((n + 15) & ~int64_t(15)) - n + rows * 8;
  return n;
}

// Past 2^24 elements the row tensors exceed what the caches keep between
// operators, and non-temporal loads measured faster (8192 x 4096: 48.1 us
// against 52.8 with plain ones); below, plain ones (2999 x 4096: 19.8 against
// 21.5).  Stores are non-temporal throughout (0-10% faster).
constexpr int64_t kCachedElements = int64_t(1) << 24;

template <int DT, int LPR, int VPL, int BLOCK, bool AHEAD = true>
void launch_rows(const NormGradArgs& a, int64_t grid, hipStream_t stream) {
  const dim3 g((unsigned)grid), b(BLOCK);
  if (a.rows > kCachedElements / a.hidden) {
    if (a.dresidual)
      norm_grad_kernel<DT, LPR, VPL, BLOCK, AHEAD, true, true><<<g, b, 0, stream>>>(a);
    else
      norm_grad_kernel<DT, LPR, VPL, BLOCK, AHEAD, false, true><<<g, b, 0, stream>>>(a);
  } else {
    if (a.dresidual)
      norm_grad_kernel<DT, LPR, VPL, BLOCK, AHEAD, true, false><<<g, b, 0, stream>>>(a);
    else
      norm_grad_kernel<DT, LPR, VPL, BLOCK, AHEAD, false, false><<<g, b, 0, stream>>>(a);
  }
}

template <int DT>
int launch_all(const NormGradArgs& a, int64_t grid, void* dweight, int dweight_dtype, hipStream_t stream) {
  if (is_general(a.hidden)) {
    float2* stats = (float2*)((char*)a.partial + ((grid * a.hidden * 4 + 15) & ~int64_t(15)));
    const unsigned rgrid = (unsigned)(a.rows < 4096 ? a.rows : 4096);
    norm_grad_stats_kernel<DT><<<dim3(rgrid), dim3(256), 0, stream>>>(a, stats);
    norm_grad_columns_kernel<DT><<<dim3((unsigned)((a.hidden + 255) / 256), (unsigned)grid), dim3(256), 0, stream>>>(
        a, stats);
    norm_grad_rows_kernel<DT><<<dim3(rgrid), dim3(256), 0, stream>>>(a, stats);
  } else {
    const Shape s = shape_of(a.hidden);
    const int key = s.lpr * 8 + s.vpl;
    switch (key) {
      case 16 * 8 + 1: launch_rows<DT, 16, 1, 256>(a, grid, stream); break;
      case 32 * 8 + 1: launch_rows<DT, 32, 1, 256>(a, grid, stream); break;
      case 64 * 8 + 1: launch_rows<DT, 64, 1, 256>(a, grid, stream); break;
      case 64 * 8 + 2: launch_rows<DT, 64, 2, 512>(a, grid, stream); break;
      case 128 * 8 + 2: launch_rows<DT, 128, 2, 256>(a, grid, stream); break;
      case 512 * 8 + 1: launch_rows<DT, 512, 1, 512>(a, grid, stream); break;
      case 256 * 8 + 3: launch_rows<DT, 256, 3, 512>(a, grid, stream); break;
      case 512 * 8 + 2: launch_rows<DT, 512, 2, 512>(a, grid, stream); break;
      case 1024 * 8 + 2: launch_rows<DT, 1024, 2, 1024, false>(a, grid, stream); break;
      default: launch_rows<DT, 1024, 4, 1024, false>(a, grid, stream); break;
    }
  }
  const dim3 wgrid((unsigned)((a.hidden + 31) / 32));
  if (dweight_dtype == HPRMS_DTYPE_FP32)
    norm_grad_weight_kernel<HPRMS_DTYPE_FP32><<<wgrid, dim3(1024), 0, stream>>>(a.partial, (int32_t)grid, a.hidden,
                                                                              dweight);
  else
    norm_grad_weight_kernel<DT><<<wgrid, dim3(1024), 0, stream>>>(a.partial, (int32_t)grid, a.hidden, dweight);
  return check_launch("rmsnorm gradient kernel");
}

int check_sizes(int64_t rows, int64_t hidden) {
  if (rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)rows);
  if (hidden < 1) return fail(HPRMS_E_INVALID, "hidden must be >= 1 (got %lld)", (long long)hidden);
  if (hidden > kMaxGradHidden)
    return fail(HPRMS_E_RANGE, "hidden %lld exceeds the supported maximum %lld", (long long)hidden,
                (long long)kMaxGradHidden);
  if (rows > (int64_t(1) << 40)) return fail(HPRMS_E_RANGE, "rows %lld exceed 2^40", (long long)rows);
  return HPRMS_OK;
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_rmsnorm_backward_workspace(int64_t rows, int64_t hidden) {
  const int rc = check_sizes(rows, hidden);
  return rc != HPRMS_OK ? rc : workspace_bytes(rows, hidden);
}

int hprms_rmsnorm_backward(void* dinput, void* dweight, const void* dout, const void* input, const void* weight,
                           const void* dresidual, void* workspace, int64_t workspace_size, int64_t rows,
                           int64_t hidden, int64_t dinput_row_stride, int64_t dout_row_stride,
                           int64_t input_row_stride, int64_t dresidual_row_stride, int dtype, int dweight_dtype,
                           double eps, hipStream_t stream) {
  if (dtype != HPRMS_DTYPE_BF16 && dtype != HPRMS_DTYPE_FP16)
    return fail(HPRMS_E_INVALID, "dtype must be HPRMS_DTYPE_BF16 or HPRMS_DTYPE_FP16 (got %d)", dtype);
  if (dweight_dtype != dtype && dweight_dtype != HPRMS_DTYPE_FP32)
    return fail(HPRMS_E_INVALID, "dweight_dtype must be dtype or HPRMS_DTYPE_FP32 (got %d)", dweight_dtype);
  const int rc = check_sizes(rows, hidden);
  if (rc != HPRMS_OK) return rc;
  if (dinput_row_stride < hidden || dout_row_stride < hidden || input_row_stride < hidden ||
      (dresidual && dresidual_row_stride < hidden))
    return fail(HPRMS_E_INVALID, "row strides must be >= hidden");
  if (!(eps >= 0.0)) return fail(HPRMS_E_INVALID, "eps must be >= 0");
  if (!extent_ok(rows, dinput_row_stride, 2, hidden) || !extent_ok(rows, dout_row_stride, 2, hidden) ||
      !extent_ok(rows, input_row_stride, 2, hidden) ||
      (dresidual && !extent_ok(rows, dresidual_row_stride, 2, hidden)))
    return fail(HPRMS_E_RANGE, "%lld rows at these row strides span more than 2^56 bytes", (long long)rows);
  if (!dweight || (rows > 0 && (!dinput || !dout || !input || !weight)))
    return fail(HPRMS_E_INVALID, "null tensor pointer");
  if ((((uintptr_t)dinput | (uintptr_t)dout | (uintptr_t)input | (uintptr_t)weight | (uintptr_t)dresidual |
        (uintptr_t)dweight) & 1) != 0 ||
      (dweight_dtype == HPRMS_DTYPE_FP32 && ((uintptr_t)dweight & 3) != 0))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  const int64_t need = workspace_bytes(rows, hidden);
  if (need > 0 && (!workspace || workspace_size < need || ((uintptr_t)workspace & 15) != 0))
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 16-byte aligned (got %lld)", (long long)need,
                (long long)workspace_size);
  // rows == 0: no partial sums, and dweight is the empty sum
  NormGradArgs a{(uint16_t*)dinput,  (const uint16_t*)dout, (const uint16_t*)input, (const uint16_t*)dresidual,
                 (const uint16_t*)weight, (float*)workspace, rows, dinput_row_stride, dout_row_stride,
                 input_row_stride, dresidual_row_stride, (int32_t)hidden, (float)eps};
  const int64_t grid = grid_of(rows, hidden);
  if (grid == 0) {
    const dim3 wgrid((unsigned)((hidden + 31) / 32));
    if (dweight_dtype == HPRMS_DTYPE_FP32)
      norm_grad_weight_kernel<HPRMS_DTYPE_FP32><<<wgrid, dim3(1024), 0, stream>>>(nullptr, 0, a.hidden, dweight);
    else
      norm_grad_weight_kernel<HPRMS_DTYPE_BF16><<<wgrid, dim3(1024), 0, stream>>>(nullptr, 0, a.hidden, dweight);
    return check_launch("rmsnorm gradient kernel");
  }
  return dtype == HPRMS_DTYPE_BF16 ? launch_all<HPRMS_DTYPE_BF16>(a, grid, dweight, dweight_dtype, stream)
                                   : launch_all<HPRMS_DTYPE_FP16>(a, grid, dweight, dweight_dtype, stream);
}

}  // extern "C"
