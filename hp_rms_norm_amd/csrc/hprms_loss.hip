// hprms_loss.hip - softmax cross entropy of rows under a vocabulary projection
// and its gradient: kernels and entry points (the mathematics: hprms_loss.h).
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_loss.h"

namespace hprms {
namespace {

// ---- the list of rows that carry a loss -----------------------------------------------
// One workgroup: `index` gets the rows whose target is not ignore_index, in
// order; with GRAD also the scale of dloss, from the largest of its finite
// magnitudes.  Without GRAD the other rows' loss and lse are set to 0.
template <bool GRAD>
__global__ __launch_bounds__(1024) void loss_rows_kernel(LossArgs a, LossMeta* meta, int32_t* index) {
  __shared__ int32_t waves[16];
  __shared__ float tops[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t count = 0;
  float top = 0.0f;
  for (int32_t r0 = 0; r0 < a.rows; r0 += 1024) {
    const int32_t row = r0 + threadIdx.x;
    const bool in = row < a.rows;
    const bool keep = in && a.target[row] != a.ignore_index;
    const uint64_t mask = __ballot(keep);
    if (lane == 0) waves[wave] = __popcll(mask);
    __syncthreads();
    int32_t before = count;
    for (int i = 0; i < 16; ++i) {
      if (i < wave) before += waves[i];
      count += waves[i];
    }
    if (keep) index[before + __popcll(mask & ((uint64_t(1) << lane) - 1))] = row;
    if constexpr (GRAD) {
      if (keep) {
        const float g = fabsf(a.dloss[row]);
        if (g < __builtin_inff()) top = fmaxf(top, g);
      }
    } else if (in && !keep) {
      a.loss[row] = 0.0f;
      a.lse[row] = 0.0f;
    }
    __syncthreads();
  }
  float scale = 1.0f;
  if constexpr (GRAD) {
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    for (int i = 0; i < 16; ++i) top = fmaxf(top, tops[i]);
    // 2^e <= top < 2^(e + 1); the scale brings it to [2^14, 2^15)
    if (top > 0.0f) {
      int e = (int)(__float_as_uint(top) >> 23) - 127;  // subnormals count as 2^-127
      e = 14 - e;
      e = e > 126 ? 126 : e < -112 ? -112 : e;
      scale = __uint_as_float((uint32_t)(e + 127) << 23);
    }
  }
  if (threadIdx.x == 0) *meta = LossMeta{count, scale, 1.0f / scale, 0};
}

// ---- forward ----------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void loss_forward_general_kernel(LossArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * kTile * kLdsRow];
  const int count = a.meta->count;
  const int n0 = a.row_from + blockIdx.y * kTile, m0 = blockIdx.x * kTile;
  if (n0 >= count) return;
  f32x4 acc[4][4];
  const Operand oa{a.weight, a.weight_stride, nullptr, a.vocab, a.width};
  const Operand ob{a.hidden, a.hidden_stride, a.index, count, a.width};
  general_tile<DT, false, false>(oa, ob, m0, n0, lds, acc);
  const int wave = threadIdx.x >> 6;
  forward_epilogue<4, 4, 2, 2>(a, acc, m0, n0, wave >> 1, wave & 1, count, blockIdx.x, (float2*)lds);
}

// Joins the tiles of RPB rows: 256 / RPB lanes per row, each over tiles in order.
template <int RPB>
__global__ __launch_bounds__(256) void loss_join_kernel(LossArgs a, int32_t tiles) {
  constexpr int S = 256 / RPB;
  __shared__ float2 lds[S][RPB];
  const int c = threadIdx.x % RPB, s = threadIdx.x / RPB;
  const int at = blockIdx.x * RPB + c;  // list position from row_from on
  const int count = a.meta->count - a.row_from;
  float top = -__builtin_inff(), sum = 0.0f;
  if (at < count) {
    for (int t = s; t < tiles; t += S) {
      const float2 o = a.partial[(int64_t)t * a.rows_at + at];
      const float m = fmaxf(top, o.x);
      const float z = m == -__builtin_inff() ? 0.0f : m;
      sum = sum * exp_neg(top - z) + o.y * exp_neg(o.x - z);
      top = m;
    }
  }
  lds[s][c] = float2{top, sum};
  __syncthreads();
  if (s != 0 || at >= count) return;
  float all = top;
  for (int i = 1; i < S; ++i) all = fmaxf(all, lds[i][c].x);
  const float z = all == -__builtin_inff() ? 0.0f : all;
  float total = 0.0f;
  for (int i = 0; i < S; ++i) total += lds[i][c].y * exp_neg(lds[i][c].x - z);
  const int row = a.index[a.row_from + at];
  const int64_t t = a.target[row];
  const float lse = all + logf(total);
  a.lse[row] = lse;
  a.loss[row] = t >= 0 && t < a.vocab ? lse - a.target_logit[a.row_from + at] : __builtin_nanf("");
}

// ---- gradient ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void loss_dz_general_kernel(LossArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * kTile * kLdsRow];
  const int count = a.meta->count;
  const int n0 = blockIdx.y * kTile, m0 = blockIdx.x * kTile;
  if (n0 >= count) return;
  f32x4 acc[4][4];
  const Operand oa{a.weight + (int64_t)a.piece_from * a.weight_stride, a.weight_stride, nullptr,
                   a.vocab - a.piece_from, a.width};
  const Operand ob{a.hidden, a.hidden_stride, a.index, count, a.width};
  general_tile<DT, false, false>(oa, ob, m0, n0, lds, acc);
  const int wave = threadIdx.x >> 6;
  dz_epilogue<DT, 4, 4>(a, acc, m0, n0, wave >> 1, wave & 1, count);
}

template <int DT>
__global__ __launch_bounds__(256) void loss_dweight_general_kernel(LossArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * kTile * kLdsRow];
  const int count = a.meta->count;
  const int m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
  f32x4 acc[4][4];
  const Operand oa{a.hidden, a.hidden_stride, a.index, a.width, count};
  const Operand ob{a.dz, a.dz_stride, nullptr, a.piece, count};
  general_tile<DT, true, true>(oa, ob, m0, n0, lds, acc);
  const int wave = threadIdx.x >> 6;
  dweight_epilogue<DT, 4, 4>(a, acc, m0, n0, wave >> 1, wave & 1);
}

template <int DT>
__global__ __launch_bounds__(256) void loss_dhidden_general_kernel(LossArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * kTile * kLdsRow];
  const int count = a.meta->count;
  const int m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
  if (n0 >= count) return;
  f32x4 acc[4][4];
  const Operand oa{a.weight + (int64_t)a.piece_from * a.weight_stride, a.weight_stride, nullptr, a.width, a.piece};
  const Operand ob{a.dz, a.dz_stride, nullptr, count, a.piece};
  general_tile<DT, true, false>(oa, ob, m0, n0, lds, acc);
  const int wave = threadIdx.x >> 6;
  dhidden_epilogue<DT, 4, 4>(a, acc, m0, n0, wave >> 1, wave & 1, count);
}

// dhidden of the rows that carry no loss
__global__ __launch_bounds__(256) void loss_zero_rows_kernel(LossArgs a) {
  for (int32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (a.target[row] != a.ignore_index) continue;
    for (int32_t i = threadIdx.x; i < a.width; i += 256) a.dhidden[(int64_t)row * a.dhidden_stride + i] = 0;
  }
}

// ---- host ---------------------------------------------------------------------------------
constexpr int64_t kMaxLossRows = int64_t(1) << 22;
constexpr int64_t kMaxLossWidth = int64_t(1) << 24;
constexpr int64_t kMaxVocab = int64_t(1) << 28;
constexpr int64_t kRowChunk = 16384;  // list positions per forward launch: bounds the partial sums
constexpr int64_t kPieceElements = int64_t(1) << 27;  // of dz per piece: 256 MiB
constexpr int64_t kMinPiece = 1024;

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }

int check_sizes(int64_t rows, int64_t width, int64_t vocab) {
  if (rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)rows);
  if (width < 1) return fail(HPRMS_E_INVALID, "hidden must be >= 1 (got %lld)", (long long)width);
  if (vocab < 1) return fail(HPRMS_E_INVALID, "vocab must be >= 1 (got %lld)", (long long)vocab);
  if (rows > kMaxLossRows || width > kMaxLossWidth || vocab > kMaxVocab)
    return fail(HPRMS_E_RANGE, "rows, hidden and vocab must be at most 2^22, 2^24 and 2^28 (got %lld, %lld, %lld)",
                (long long)rows, (long long)width, (long long)vocab);
  return HPRMS_OK;
}

// Offsets of the workspace's parts, bytes.
struct ForwardPlan {
  int64_t index, target_logit, partial, total;
  int64_t rows_at, tiles;
};

ForwardPlan forward_plan(int64_t rows, int64_t vocab) {
  ForwardPlan p;
  p.rows_at = min64(rows, kRowChunk);
  p.tiles = (vocab + kTile - 1) / kTile;
  p.index = 256;
  p.target_logit = p.index + round_up(rows * 4, 256);
  p.partial = p.target_logit + round_up(rows * 4, 256);
  p.total = p.partial + p.tiles * p.rows_at * 8;
  return p;
}

struct BackwardPlan {
  int64_t index, dz, sum, total;
  int64_t piece, pieces, dz_rows;
};

BackwardPlan backward_plan(int64_t rows, int64_t width, int64_t vocab) {
  BackwardPlan p;
  p.dz_rows = round_up(rows, kTile);
  const int64_t whole = round_up(vocab, kTile);
  p.piece = kPieceElements / (p.dz_rows > 0 ? p.dz_rows : kTile) / kTile * kTile;
  if (p.piece < kMinPiece) p.piece = kMinPiece;
  if (p.piece > whole) p.piece = whole;
  p.pieces = (vocab + p.piece - 1) / p.piece;
  p.index = 256;
  p.dz = p.index + round_up(rows * 4, 256);
  p.sum = p.dz + p.dz_rows * p.piece * 2;
  p.total = p.sum + (p.pieces > 1 ? rows * width * 4 : 0);
  return p;
}

bool aligned_to(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_common(const void* hidden, const void* weight, const int64_t* target, int64_t rows, int64_t width,
                 int64_t vocab, int64_t hidden_stride, int64_t weight_stride, int dtype) {
  if (dtype != HPRMS_DTYPE_BF16 && dtype != HPRMS_DTYPE_FP16)
    return fail(HPRMS_E_INVALID, "dtype must be HPRMS_DTYPE_BF16 or HPRMS_DTYPE_FP16 (got %d)", dtype);
  const int rc = check_sizes(rows, width, vocab);
  if (rc != HPRMS_OK) return rc;
  if (hidden_stride < width || weight_stride < width)
    return fail(HPRMS_E_INVALID, "row strides must be >= hidden");
  if (!extent_ok(rows, hidden_stride, 2, width) || !extent_ok(vocab, weight_stride, 2, width))
    return fail(HPRMS_E_RANGE, "the rows at these row strides span more than 2^56 bytes");
  if (rows > 0 && (!hidden || !weight || !target)) return fail(HPRMS_E_INVALID, "null tensor pointer");
  if (!aligned_to(hidden, 2) || !aligned_to(weight, 2) || !aligned_to(target, 8))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  return HPRMS_OK;
}

int check_workspace(const void* workspace, int64_t size, int64_t need) {
  if (!workspace || size < need || !aligned_to(workspace, 256))
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 256-byte aligned (got %lld)", (long long)need,
                (long long)size);
  return HPRMS_OK;
}

template <int DT>
int run_forward(LossArgs a, const ForwardPlan& p, LossMeta* meta, int32_t* index, hipStream_t stream) {
  loss_rows_kernel<false><<<dim3(1), dim3(1024), 0, stream>>>(a, meta, index);
  for (int64_t from = 0; from < a.rows; from += p.rows_at) {
    a.row_from = (int32_t)from;
    a.rows_at = (int32_t)p.rows_at;
    const int64_t here = min64(p.rows_at, a.rows - from);
    loss_forward_general_kernel<DT><<<dim3((unsigned)p.tiles, (unsigned)((here + kTile - 1) / kTile)), dim3(256), 0,
                                      stream>>>(a);
    if (here < 256)
      loss_join_kernel<1><<<dim3((unsigned)here), dim3(256), 0, stream>>>(a, (int32_t)p.tiles);
    else
      loss_join_kernel<16><<<dim3((unsigned)((here + 15) / 16)), dim3(256), 0, stream>>>(a, (int32_t)p.tiles);
  }
  return check_launch("cross entropy kernel");
}

template <int DT>
int run_backward(LossArgs a, const BackwardPlan& p, LossMeta* meta, int32_t* index, hipStream_t stream) {
  loss_rows_kernel<true><<<dim3(1), dim3(1024), 0, stream>>>(a, meta, index);
  if (a.rows > 0)
    loss_zero_rows_kernel<<<dim3((unsigned)min64(a.rows, 4096)), dim3(256), 0, stream>>>(a);
  const unsigned row_tiles = (unsigned)((a.rows + kTile - 1) / kTile);
  const unsigned width_tiles = (unsigned)((a.width + kTile - 1) / kTile);
  for (int64_t i = 0; i < p.pieces; ++i) {
    a.piece_from = (int32_t)(i * p.piece);
    a.piece = (int32_t)min64(p.piece, a.vocab - a.piece_from);
    a.first_piece = i == 0;
    a.last_piece = i + 1 == p.pieces;
    const unsigned tiles = (unsigned)((a.piece + kTile - 1) / kTile);
    if (row_tiles > 0) loss_dz_general_kernel<DT><<<dim3(tiles, row_tiles), dim3(256), 0, stream>>>(a);
    loss_dweight_general_kernel<DT><<<dim3(width_tiles, tiles), dim3(256), 0, stream>>>(a);
    if (row_tiles > 0) loss_dhidden_general_kernel<DT><<<dim3(width_tiles, row_tiles), dim3(256), 0, stream>>>(a);
  }
  return check_launch("cross entropy gradient kernel");
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_linear_cross_entropy_workspace(int64_t rows, int64_t hidden, int64_t vocab) {
  const int rc = check_sizes(rows, hidden, vocab);
  return rc != HPRMS_OK ? rc : forward_plan(rows, vocab).total;
}

int hprms_linear_cross_entropy(float* loss, float* lse, const void* hidden, const void* weight, const int64_t* target,
                               void* workspace, int64_t workspace_size, int64_t rows, int64_t hidden_size,
                               int64_t vocab, int64_t hidden_row_stride, int64_t weight_row_stride,
                               int64_t ignore_index, int dtype, hipStream_t stream) {
  int rc = check_common(hidden, weight, target, rows, hidden_size, vocab, hidden_row_stride, weight_row_stride, dtype);
  if (rc != HPRMS_OK) return rc;
  if (rows == 0) return HPRMS_OK;
  if (!loss || !lse || !aligned_to(loss, 4) || !aligned_to(lse, 4))
    return fail(HPRMS_E_INVALID, "null or misaligned tensor pointer (loss, lse)");
  const ForwardPlan p = forward_plan(rows, vocab);
  rc = check_workspace(workspace, workspace_size, p.total);
  if (rc != HPRMS_OK) return rc;
  char* ws = (char*)workspace;
  LossArgs a = {};
  a.hidden = (const uint16_t*)hidden;
  a.weight = (const uint16_t*)weight;
  a.target = target;
  a.meta = (const LossMeta*)ws;
  a.index = (const int32_t*)(ws + p.index);
  a.hidden_stride = hidden_row_stride;
  a.weight_stride = weight_row_stride;
  a.ignore_index = ignore_index;
  a.rows = (int32_t)rows;
  a.width = (int32_t)hidden_size;
  a.vocab = (int32_t)vocab;
  a.loss = loss;
  a.lse = lse;
  a.target_logit = (float*)(ws + p.target_logit);
  a.partial = (float2*)(ws + p.partial);
  return dtype == HPRMS_DTYPE_BF16
             ? run_forward<HPRMS_DTYPE_BF16>(a, p, (LossMeta*)ws, (int32_t*)(ws + p.index), stream)
             : run_forward<HPRMS_DTYPE_FP16>(a, p, (LossMeta*)ws, (int32_t*)(ws + p.index), stream);
}

int64_t hprms_linear_cross_entropy_backward_workspace(int64_t rows, int64_t hidden, int64_t vocab) {
  const int rc = check_sizes(rows, hidden, vocab);
  return rc != HPRMS_OK ? rc : backward_plan(rows, hidden, vocab).total;
}

int hprms_linear_cross_entropy_backward(void* dhidden, void* dweight, const float* dloss, const void* hidden,
                                        const void* weight, const int64_t* target, const float* lse, void* workspace,
                                        int64_t workspace_size, int64_t rows, int64_t hidden_size, int64_t vocab,
                                        int64_t dhidden_row_stride, int64_t dweight_row_stride,
                                        int64_t hidden_row_stride, int64_t weight_row_stride, int64_t ignore_index,
                                        int dtype, hipStream_t stream) {
  int rc = check_common(hidden, weight, target, rows, hidden_size, vocab, hidden_row_stride, weight_row_stride, dtype);
  if (rc != HPRMS_OK) return rc;
  if (dhidden_row_stride < hidden_size || dweight_row_stride < hidden_size)
    return fail(HPRMS_E_INVALID, "row strides must be >= hidden");
  if (!extent_ok(rows, dhidden_row_stride, 2, hidden_size) || !extent_ok(vocab, dweight_row_stride, 2, hidden_size))
    return fail(HPRMS_E_RANGE, "the rows at these row strides span more than 2^56 bytes");
  if (!dweight || (rows > 0 && (!dhidden || !dloss || !lse)))
    return fail(HPRMS_E_INVALID, "null tensor pointer");
  if (!aligned_to(dweight, 2) || !aligned_to(dhidden, 2) || !aligned_to(dloss, 4) || !aligned_to(lse, 4))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  const BackwardPlan p = backward_plan(rows, hidden_size, vocab);
  rc = check_workspace(workspace, workspace_size, p.total);
  if (rc != HPRMS_OK) return rc;
  char* ws = (char*)workspace;
  LossArgs a = {};
  a.hidden = (const uint16_t*)hidden;
  a.weight = (const uint16_t*)weight;
  a.target = target;
  a.meta = (const LossMeta*)ws;
  a.index = (const int32_t*)(ws + p.index);
  a.hidden_stride = hidden_row_stride;
  a.weight_stride = weight_row_stride;
  a.ignore_index = ignore_index;
  a.rows = (int32_t)rows;
  a.width = (int32_t)hidden_size;
  a.vocab = (int32_t)vocab;
  a.lse = const_cast<float*>(lse);
  a.dloss = dloss;
  a.dz = (uint16_t*)(ws + p.dz);
  a.dz_stride = p.piece;
  a.dhidden = (uint16_t*)dhidden;
  a.dhidden_stride = dhidden_row_stride;
  a.dweight = (uint16_t*)dweight;
  a.dweight_stride = dweight_row_stride;
  a.sum = (float*)(ws + p.sum);
  return dtype == HPRMS_DTYPE_BF16
             ? run_backward<HPRMS_DTYPE_BF16>(a, p, (LossMeta*)ws, (int32_t*)(ws + p.index), stream)
             : run_backward<HPRMS_DTYPE_FP16>(a, p, (LossMeta*)ws, (int32_t*)(ws + p.index), stream);
}

}  // extern "C"
