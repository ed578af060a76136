// hprms_loss.hip - softmax cross entropy of rows under a vocabulary projection
// and its gradient: kernels and entry points (the mathematics: hprms_loss.h).
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_loss.h"

namespace hprms {
namespace {

// The packed rows transposed, for dweight: its products sum over the rows, and
// of two operands that lie across the sum (k outer) one costs the matrix cores
// 7% (4096 x 32768 x 4096 tiles: 1340 TFLOP/s with hidden k contiguous, 1250
// with both k outer).  One workgroup turns 64 x 64.
__global__ __launch_bounds__(256) void loss_turn_kernel(LossArgs a, uint16_t* turned) {
  __shared__ uint16_t tile[64][66];  // 33 banks a row
  const int count = a.meta->count;
  const int n0 = blockIdx.x * 64, w0 = blockIdx.y * 64;
  if (n0 >= count) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = threadIdx.x + i * 256, n = e >> 3, w = (e & 7) * 8;
    u32x4 v = {0, 0, 0, 0};
    if (n0 + n < count) v = *(const u32x4*)(a.packed + (int64_t)(n0 + n) * a.packed_width + w0 + w);
#pragma unroll
    for (int j = 0; j < 4; ++j) *(uint32_t*)&tile[n][w + 2 * j] = v[j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = threadIdx.x + i * 256, w = e >> 3, n = (e & 7) * 8;
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = tile[n + 2 * j][w] | (uint32_t)tile[n + 2 * j + 1][w] << 16;
    *(u32x4*)(turned + (int64_t)(w0 + w) * a.turned_stride + n0 + n) = v;
  }
}

// A piece of a weight whose rows the products cannot read in place (an odd
// width, stride or alignment), packed likewise.
__global__ __launch_bounds__(256) void loss_pack_weight_kernel(const uint16_t* weight, int64_t stride, int32_t rows,
                                                               int32_t width, int32_t packed_width,
                                                               uint16_t* packed) {
  for (int32_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const uint16_t* from = weight + (int64_t)row * stride;
    uint16_t* to = packed + (int64_t)row * packed_width;
    for (int32_t i = threadIdx.x * 8; i < packed_width; i += 256 * 8) *(u32x4*)(to + i) = load_some(from + i, width - i);
  }
}

// ---- operands -----------------------------------------------------------------------------
// the piece's weight rows from row m on: k contiguous (z) ...
__device__ __forceinline__ Operand weight_rows(const LossArgs& a, int m) {
  return {a.weight + (int64_t)m * a.weight_stride,
          ((int64_t)(a.piece - 1 - m) * a.weight_stride + a.weight_width) * 2, a.weight_stride};
}
// ... or as the summed index, from entry k on, hidden elements from m on
__device__ __forceinline__ Operand weight_columns(const LossArgs& a, int k, int m) {
  return {a.weight + (int64_t)k * a.weight_stride + m,
          ((int64_t)(a.piece - 1 - k) * a.weight_stride + a.weight_width - m) * 2, a.weight_stride};
}
__device__ __forceinline__ Operand packed_rows(const LossArgs& a, int n, int count) {
  return {a.packed + (int64_t)n * a.packed_width, (int64_t)(count - n) * a.packed_width * 2, a.packed_width};
}
__device__ __forceinline__ Operand packed_columns(const LossArgs& a, int k, int m, int count) {
  return {a.packed + (int64_t)k * a.packed_width + m, ((int64_t)(count - k) * a.packed_width - m) * 2, a.packed_width};
}
__device__ __forceinline__ Operand turned_rows(const LossArgs& a, int m, int k) {
  return {a.turned + (int64_t)m * a.turned_stride + k, ((int64_t)(a.packed_width - m) * a.turned_stride - k) * 2,
          a.turned_stride};
}
__device__ __forceinline__ Operand dz_rows(const LossArgs& a, int n, int v, int count) {
  return {a.dz + (int64_t)n * a.dz_stride + v, ((int64_t)(count - n) * a.dz_stride - v) * 2, a.dz_stride};
}
__device__ __forceinline__ Operand dz_columns(const LossArgs& a, int v, int k, int count) {
  return {a.dz + (int64_t)k * a.dz_stride + v, ((int64_t)(count - k) * a.dz_stride - v) * 2, a.dz_stride};
}

// ---- forward ----------------------------------------------------------------------------
template <class P, int DT>
__global__ __launch_bounds__(P::NW * 64) void loss_forward_kernel(LossArgs a, int group) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[P::LDS_BYTES / 2];
  const int count = a.meta->count;
  const int here = min(count - a.row_from, a.rows_at);
  int m, n;
  if (here <= 0 || !tile_of(blockIdx.x, a.vocab_tiles, (here + P::NT - 1) / P::NT, group, &m, &n)) return;
  const int m0 = m * P::MT, n0 = a.row_from + n * P::NT;
  const int wave = threadIdx.x >> 6, end = min(count, a.row_from + a.rows_at);
  int t[P::NI];
  load_targets<P::NI>(a, n0, wave % P::WN, end, t);
  f32x4 acc[P::MI][P::NI];
  P::run(weight_rows(a, m0), packed_rows(a, n0, count), a.width, lds, acc);
  // (a SumProduct's waves all hold the whole tile, and all do the same)
  forward_epilogue<P::MI, P::NI, P::WM, P::WN>(a, acc, t, m0, n0, wave / P::WN % P::WM, wave % P::WN, end,
                                               a.tile_from + m, (float2*)lds);
}

// Two maxima with their sums of exponentials relative to them, as one.
__device__ __forceinline__ float2 join(float2 s, float2 o) {
  const float top = fmaxf(s.x, o.x);
  const float at = top == -__builtin_inff() ? 0.0f : top;
  return {top, s.y * exp_neg(s.x - at) + o.y * exp_neg(o.x - at)};
}

// Joins the tiles of RPB rows: 256 / RPB lanes a row, each over every so many
// tiles, then the lanes.
template <int RPB>
__global__ __launch_bounds__(256) void loss_join_kernel(LossArgs a, int32_t tiles) {
  constexpr int S = 256 / RPB, U = 8;
  __shared__ float2 lds[4][RPB];
  const int c = threadIdx.x % RPB, s = threadIdx.x / RPB;
  const int at = blockIdx.x * RPB + c;  // list position from row_from on
  const bool live = at < a.meta->count - a.row_from;
  const float2 none = {-__builtin_inff(), 0.0f};
  float2 all = none;
  for (int t = s; t < tiles; t += S * U) {
    float2 o[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      o[i] = live && t + i * S < tiles ? a.partial[(int64_t)(t + i * S) * a.rows_at + at] : none;
    float top = all.x;
#pragma unroll
    for (int i = 0; i < U; ++i) top = fmaxf(top, o[i].x);
    const float z = top == -__builtin_inff() ? 0.0f : top;
    float sum = all.y * exp_neg(all.x - z);
#pragma unroll
    for (int i = 0; i < U; ++i) sum += o[i].y * exp_neg(o[i].x - z);
    all = {top, sum};
  }
#pragma unroll
  for (int m = RPB; m < 64; m <<= 1) all = join(all, {__shfl_xor(all.x, m), __shfl_xor(all.y, m)});
  if ((threadIdx.x & 63) < RPB) lds[threadIdx.x >> 6][c] = all;
  __syncthreads();
  if (s != 0 || !live) return;
  for (int i = 1; i < 4; ++i) all = join(all, lds[i][c]);
  const int row = a.index[a.row_from + at];
  const int64_t t = a.target[row];
  const float lse = all.x + logf(all.y);
  a.lse[row] = lse;
  a.loss[row] = t >= 0 && t < a.vocab ? lse - a.target_logit[a.row_from + at] : __builtin_nanf("");
}

// ---- gradient ---------------------------------------------------------------------------
// LDS of a kernel whose tile leaves through it
template <class P>
constexpr int kLdsOut = P::LDS_BYTES > kTileOutBytes<P> ? P::LDS_BYTES : kTileOutBytes<P>;

template <class P, int DT>
__global__ __launch_bounds__(P::NW * 64) void loss_dz_kernel(LossArgs a, int group) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[P::LDS_BYTES / 2];
  const int count = a.meta->count;
  int m, n;
  if (!tile_of(blockIdx.x, a.vocab_tiles, (count + P::NT - 1) / P::NT, group, &m, &n)) return;
  const int m0 = m * P::MT, n0 = n * P::NT;
  DzColumns<P> columns;
  columns.load(a, n0, (threadIdx.x >> 6) % P::WN, count);
  f32x4 acc[P::MI][P::NI];
  P::run(weight_rows(a, m0), packed_rows(a, n0, count), a.width, lds, acc);
  if (P::NW > P::WM * P::WN && threadIdx.x >= P::WM * P::WN * 64) return;  // a SumProduct's first wave has it all
  dz_epilogue<P, DT>(a, acc, columns, m0, n0, count);
}

// Splits of a product's summed entries over workgroups, where it has fewer tiles
// than `slots` (the workgroups that run at once): as many as fill them, of at
// least 256 entries each, and `most` at the most.  The count of listed rows is
// known on the device alone, so kernels and host compute this where they are.
struct Splits {
  int32_t count, span;
};
__host__ __device__ inline Splits splits_of(int32_t tiles, int32_t slots, int32_t depth, int32_t most) {
  int32_t n = slots / (tiles > 0 ? tiles : 1);
  if (n > depth / 256) n = depth / 256;
  if (n > most) n = most;
  if (n < 1) n = 1;
  const int32_t span = ((depth + n - 1) / n + 63) / 64 * 64;
  return {span > 0 ? (depth + span - 1) / span : 1, span > 0 ? span : 64};
}

__device__ __forceinline__ Splits weight_splits(const LossArgs& a, int count) {
  const Splits sp = splits_of(((a.piece + 127) / 128) * ((a.width + 127) / 128), a.slots, count, a.weight_most);
  return {sp.count > 0 ? sp.count : 1, sp.span};
}

template <class P, int DT>
__global__ __launch_bounds__(P::NW * 64) void loss_dweight_kernel(LossArgs a, int group) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[kLdsOut<P> / 2];
  const int count = a.meta->count;
  const Splits sp = a.weight_sum ? weight_splits(a, count) : Splits{1, (count + 63) & ~63};
  int m, ns;
  if (!tile_of(blockIdx.x, a.width_tiles, a.vocab_tiles * sp.count, group, &m, &ns)) return;
  const int n = ns % a.vocab_tiles, split = ns / a.vocab_tiles, from = split * sp.span;
  const int m0 = m * P::MT, n0 = n * P::NT;
  f32x4 acc[P::MI][P::NI];
  // rows past the count are out of range or, in `turned`, zeros, so the depth may be rounded up to whole chunks
  Operand hidden;
  if constexpr (P::AKO)
    hidden = packed_columns(a, from, m0, count);
  else
    hidden = turned_rows(a, m0, from);
  P::run(hidden, dz_columns(a, n0, from, count), max(0, min(sp.span, (count - from + 7) & ~7)), lds, acc);
  if (sp.count == 1) {
    dweight_epilogue<P, DT>(a, acc, m0, n0, lds);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / P::WN, wn = wave % P::WN;
  float* to = a.weight_sum + (int64_t)split * ((a.piece + 127) & ~127) * a.packed_width;
#pragma unroll
  for (int ni = 0; ni < P::NI; ++ni)
#pragma unroll
    for (int mi = 0; mi < P::MI; ++mi) {
      const int v = n0 + (wn * P::NI + ni) * 16 + (lane & 15), i = m0 + (wm * P::MI + mi) * 16 + (lane >> 4) * 4;
      if (v < a.piece && i < a.packed_width) *(f32x4*)(to + (int64_t)v * a.packed_width + i) = acc[mi][ni];
    }
}

// A row's sum of its shares, elements i ... i + 3.
__device__ __forceinline__ f32x4 sum_shares(const float* from, int64_t step, int splits) {
  f32x4 d = {0, 0, 0, 0};
  constexpr int U = 8;  // loads on their way at once
  for (int s = 0; s < splits; s += U) {
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = f32x4{0, 0, 0, 0};
      if (s + u < splits) v[u] = *(const f32x4*)(from + (s + u) * step);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) d += v[u];
  }
  return d;
}

// ... scaled back and rounded, the first `left` of the four
template <int DT>
__device__ __forceinline__ void store_sum(uint16_t* to, f32x4 d, float unscale, int left) {
  const float o[4] = {d[0] * unscale, d[1] * unscale, d[2] * unscale, d[3] * unscale};
  store_four<DT>(to, o, left);
}

// dweight from its shares, if it has any
template <int DT>
__global__ __launch_bounds__(256) void loss_dweight_sum_kernel(LossArgs a) {
  const int splits = weight_splits(a, a.meta->count).count;
  if (splits == 1) return;
  const float unscale = a.meta->unscale;
  const int64_t step = (int64_t)((a.piece + 127) & ~127) * a.packed_width;
  for (int32_t v = blockIdx.x; v < a.piece; v += gridDim.x)
    for (int32_t i = threadIdx.x * 4; i < a.width; i += 1024)
      store_sum<DT>(a.dweight + ((int64_t)a.piece_from + v) * a.dweight_stride + i,
                    sum_shares(a.weight_sum + (int64_t)v * a.packed_width + i, step, splits), unscale, a.width - i);
}

template <class P, int DT>
__global__ __launch_bounds__(P::NW * 64) void loss_dhidden_product_kernel(LossArgs a, int group) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[P::LDS_BYTES / 2];
  const int count = a.meta->count;
  const int row_tiles = (count + P::NT - 1) / P::NT;
  const Splits sp = splits_of(a.width_tiles * row_tiles, a.slots, a.piece_size, a.most_splits);
  int m, ns;
  if (!tile_of(blockIdx.x, a.width_tiles, row_tiles * sp.count, group, &m, &ns)) return;
  const int n = ns % row_tiles, split = ns / row_tiles, span = sp.span;
  const int m0 = m * P::MT, n0 = n * P::NT;
  const int from = split * span;
  // dz holds zeros past the piece up to a tile's end, so the depth may be rounded up to whole chunks
  const int depth = max(0, min(span, (a.piece - from + 7) & ~7));
  f32x4 acc[P::MI][P::NI];
  P::run(weight_columns(a, from, m0), dz_rows(a, n0, from, count), depth, lds, acc);
  const int wave = threadIdx.x >> 6;
  dhidden_epilogue<DT, P::MI, P::NI>(a, acc, m0, n0, wave / P::WN, wave % P::WN, count, split);
}

// dhidden from its shares
template <int DT>
__global__ __launch_bounds__(256) void loss_dhidden_kernel(LossArgs a, int tile_rows) {
  const int count = a.meta->count;
  const int splits = splits_of(a.width_tiles * ((count + tile_rows - 1) / tile_rows), a.slots, a.piece_size,
                               a.most_splits).count;
  const float unscale = a.meta->unscale;
  const int64_t step = (int64_t)count * a.packed_width;
  for (int32_t n = blockIdx.x; n < count; n += gridDim.x) {
    const int32_t row = a.index[n];
    for (int32_t i = (blockIdx.y * 256 + threadIdx.x) * 4; i < a.width; i += gridDim.y * 1024)
      store_sum<DT>(a.dhidden + (int64_t)row * a.dhidden_stride + i,
                    sum_shares(a.sum + (int64_t)n * a.packed_width + i, step, splits), unscale, a.width - i);
  }
}

// ---- host ---------------------------------------------------------------------------------
constexpr int64_t kMaxLossRows = int64_t(1) << 22;
constexpr int64_t kMaxLossWidth = int64_t(1) << 20;
constexpr int64_t kMaxVocab = int64_t(1) << 28;
constexpr int64_t kRowChunk = 16384;  // list positions per forward launch: bounds the partial sums
// tiles per forward launch, a multiple of 8: with up to 512 lanes each they stay
// below the 2^32 work-items that a launch may hold
constexpr int64_t kForwardTiles = (int64_t(1) << 23) - 8;
constexpr int64_t kPieceElements = int64_t(1) << 27;  // of dz, and of a packed weight, per piece: 256 MiB
constexpr int64_t kHiddenTile = 256;  // hidden elements of a dhidden tile
constexpr int64_t kPieceUnit = 256;   // pieces are whole tiles of every kernel
// a tile's 256 rows at this stride stay within a buffer access's 31-bit offset
constexpr int64_t kMaxWeightStride = int64_t(1) << 21;

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t ceil_div(int64_t v, int64_t m) { return (v + m - 1) / m; }
int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }
int64_t max64(int64_t a, int64_t b) { return a > b ? a : b; }
bool aligned_to(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_sizes(int64_t rows, int64_t width, int64_t vocab) {
  if (rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)rows);
  if (width < 1) return fail(HPRMS_E_INVALID, "hidden must be >= 1 (got %lld)", (long long)width);
  if (vocab < 1) return fail(HPRMS_E_INVALID, "vocab must be >= 1 (got %lld)", (long long)vocab);
  if (rows > kMaxLossRows || width > kMaxLossWidth || vocab > kMaxVocab)
    return fail(HPRMS_E_RANGE, "rows, hidden and vocab must be at most 2^22, 2^20 and 2^28 (got %lld, %lld, %lld)",
                (long long)rows, (long long)width, (long long)vocab);
  return HPRMS_OK;
}

// The products read the weight's rows in place where 16-byte loads at 16-byte
// boundaries cover them; otherwise a piece at a time is packed first.
bool weight_in_place(const void* weight, int64_t stride, int64_t width) {
  return aligned_to(weight, 16) && stride % 8 == 0 && width % 8 == 0 && stride <= kMaxWeightStride;
}

int64_t packed_width_of(int64_t width) { return round_up(width, 64); }

// vocabulary rows of a packed piece
int64_t packed_piece(int64_t width, int64_t vocab) {
  const int64_t p = max64(kPieceElements / packed_width_of(width) / kPieceUnit * kPieceUnit, kPieceUnit);
  return min64(p, round_up(vocab, kPieceUnit));
}

// Tiles of z, vocabulary rows x list positions, by the number of rows: 128 x 16
// and 128 x 64 (the weight's bytes bound these: 131072 x 4096 in 185 us, 5.8
// TB/s, up to 64 rows), 256 x 128, 256 x 256; 64 x 16 and 64 x 64 where 128
// vocabulary rows would leave a CU fewer than two workgroups (14814 x 6656, 23
// rows: 45 us, 55 with 128 x 64); 16 x 16, whose waves share the sum, up to one
// workgroup a CU (1361 x 4544, 1 row: 9.0 us, 64 x 16 21; beyond, 17839 x 768, 6
// rows, 14.4 against 8.5); and 128 x 128 where 256 x 256 would leave half of the
// CUs without a tile.  In batch-invariant mode always 256 x 256: the shapes sum a
// row's exponentials, and 16 x 16 its logits, in other orders, which shows in the
// last bits of its lse.
enum LogitTile { kTile16Sum, kTile16Short, kTile64Short, kTile16, kTile64, kTileSmall, kTile128, kTile256 };
LogitTile logit_tile(int64_t rows, int64_t vocab, bool invariant) {
  if (invariant) return kTile256;
  if (rows <= 64) {
    if (rows <= 16 && ceil_div(vocab, 16) <= current_cus()) return kTile16Sum;
    if (ceil_div(vocab, 128) < 2 * (int64_t)current_cus()) return rows <= 16 ? kTile16Short : kTile64Short;
    return rows <= 16 ? kTile16 : kTile64;
  }
  if (2 * ceil_div(vocab, 256) * ceil_div(rows, 256) <= current_cus()) return kTileSmall;
  return rows <= 128 ? kTile128 : kTile256;
}
int64_t logit_vocab_rows(LogitTile t) {
  return t == kTile16Sum ? 16 : t <= kTile64Short ? 64 : t <= kTileSmall ? 128 : 256;
}
int64_t logit_rows(LogitTile t) {
  return t <= kTile16Short || t == kTile16   ? 16
         : t == kTile64Short || t == kTile64 ? 64
         : t == kTile256                     ? 256
                                             : 128;
}

// Offsets of the workspace's parts, bytes.  A call reads the batch-invariant
// mode once, into its plan.
struct ForwardPlan {
  int64_t index, target_logit, packed, weight, partial, total;
  int64_t rows_at, tiles, piece;
  LogitTile tile;
  bool invariant;
};

ForwardPlan forward_plan(int64_t rows, int64_t width, int64_t vocab, bool in_place, bool invariant) {
  ForwardPlan p;
  p.invariant = invariant;
  p.tile = logit_tile(rows, vocab, invariant);
  p.piece = in_place ? round_up(vocab, kPieceUnit) : packed_piece(width, vocab);
  p.tiles = ceil_div(vocab, logit_vocab_rows(p.tile));
  p.rows_at = min64(min64(rows, kRowChunk), kForwardTiles / p.tiles * logit_rows(p.tile));
  p.index = 256;
  p.target_logit = p.index + round_up(rows * 4, 256);
  p.packed = p.target_logit + round_up(rows * 4, 256);
  p.weight = p.packed + rows * packed_width_of(width) * 2;
  p.partial = p.weight + (in_place ? 0 : p.piece * packed_width_of(width) * 2);
  p.total = p.partial + p.tiles * p.rows_at * 8;
  return p;
}

struct BackwardPlan {
  int64_t index, packed, turned, weight, dz, sum, total;
  int64_t turned_stride;
  int64_t piece, pieces, dz_rows, row_tiles, width_tiles, slots, most_splits;
  int64_t weight_sum, weight_most;
  bool shares, few;
  LogitTile tile;
};

BackwardPlan backward_plan(int64_t rows, int64_t width, int64_t vocab, bool in_place, bool invariant) {
  BackwardPlan p;
  p.tile = logit_tile(rows, vocab, invariant);
  p.dz_rows = round_up(max64(rows, 1), logit_rows(p.tile));
  p.piece = max64(kPieceElements / max64(p.dz_rows, 256) / kPieceUnit * kPieceUnit, 4 * kPieceUnit);
  p.piece = min64(p.piece, round_up(vocab, kPieceUnit));
  if (!in_place) p.piece = min64(p.piece, packed_piece(width, vocab));
  p.pieces = ceil_div(vocab, p.piece);
  p.width_tiles = ceil_div(width, kHiddenTile);
  const int64_t row_tiles = ceil_div(max64(rows, 1), logit_rows(p.tile));
  p.slots = (int64_t)current_cus() * (p.tile == kTile256 ? 1 : 2);
  // with fewer listed rows there are more splits, of fewer rows: count * splits
  // stays within what a slot's tile holds each, or within one share of all rows
  p.most_splits = max64(1, min64(p.slots / p.width_tiles, p.piece / 256));
  const int64_t sum_rows = max64(rows, p.most_splits > 1 ? p.slots / p.width_tiles * logit_rows(p.tile) : 0);
  const bool shares = p.pieces > 1 || p.most_splits > 1;
  // dweight in tiles of 128 x 128, which run four to a CU, where the sums over
  // the rows are short (128 rows of 131072 x 4096: 331 us, 256 x 256 430) or 256 x
  // 256 would leave CUs without a tile; where even these do, the rows are split
  p.few = rows <= 128 || ceil_div(p.piece, 256) * ceil_div(width, 256) < current_cus();
  p.index = 256;
  p.packed = p.index + round_up(rows * 4, 256);
  p.turned_stride = round_up(rows, 64);
  p.turned = p.packed + round_up(rows * packed_width_of(width) * 2, 256);
  p.weight = p.turned + (p.few ? 0 : p.turned_stride * packed_width_of(width) * 2);
  p.dz = p.weight + (in_place ? 0 : p.piece * packed_width_of(width) * 2);
  p.sum = p.dz + p.dz_rows * p.piece * 2;
  p.total = p.sum + (shares ? sum_rows * packed_width_of(width) * 4 : 0);
  p.row_tiles = row_tiles;
  p.shares = shares;
  p.weight_most = 1;
  if (p.few && p.pieces == 1)
    p.weight_most = max64(1, min64(p.slots / (ceil_div(vocab, 128) * ceil_div(width, 128)), rows / 256));
  p.weight_sum = round_up(p.total, 256);
  if (p.weight_most > 1) p.total = p.weight_sum + p.weight_most * round_up(vocab, 128) * packed_width_of(width) * 4;
  return p;
}

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

// Tiles of the products over the hidden index (z: A and B k contiguous) and over
// the vocabulary (dhidden: A k outer).  An operand that lies k outer takes more
// LDS instructions a fragment, so its side of a wave's part is the short one.
template <int DT, bool AKO>
struct Tiles {
  typedef std::conditional_t<AKO, Product<DT, 256, 16, 4, 1, 32, 4, true, false>,
                             Product<DT, 128, 16, 4, 1, 64, 4, false, false>> T16;
  typedef std::conditional_t<AKO, Product<DT, 256, 64, 4, 1, 32, 4, true, false>,
                             Product<DT, 128, 64, 4, 1, 64, 3, false, false>> T64;
  typedef SumProduct<DT, 1, 1, 4, 6> T16Sum;
  typedef Product<DT, 64, 16, 4, 1, 64, 6, false, false> T16Short;
  typedef Product<DT, 64, 64, 4, 1, 64, 5, false, false> T64Short;
  typedef Product<DT, 128, 128, 2, 2, 64, 2, false, false> Small;
  typedef Product<DT, 256, 128, 4, 2, 32, 3, AKO, false> T128;
  typedef RingProduct<DT, AKO, false, AKO ? 4 : 2> T256;
};

// workgroups of `tiles` tiles, for tile_of
unsigned grid_of(int64_t tiles) { return (unsigned)round_up(tiles, 8); }

template <class P, int DT>
void launch_forward(LossArgs a, int64_t here, hipStream_t stream) {
  a.vocab_tiles = (int32_t)ceil_div(a.piece, P::MT);
  const int64_t tiles = a.vocab_tiles * ceil_div(here, P::NT);
  loss_forward_kernel<P, DT><<<dim3(grid_of(tiles)), dim3(P::NW * 64), 0, stream>>>(a, 4);
}

// what a call's pieces of the vocabulary share: the piece's rows, packed if need be
struct Weight {
  const uint16_t* base;
  int64_t stride;
  uint16_t* packed;  // null: in place
};

void take_piece(LossArgs& a, const Weight& w, int64_t from, int64_t piece, hipStream_t stream) {
  a.piece_from = (int32_t)from;
  a.piece = (int32_t)min64(piece, a.vocab - from);
  const uint16_t* rows = w.base + from * w.stride;
  if (!w.packed) {
    a.weight = rows;
    a.weight_stride = (int32_t)w.stride;
    a.weight_width = a.width;
    return;
  }
  loss_pack_weight_kernel<<<dim3((unsigned)min64(a.piece, 8192)), dim3(256), 0, stream>>>(
      rows, w.stride, a.piece, a.width, a.packed_width, w.packed);
  a.weight = w.packed;
  a.weight_stride = a.packed_width;
  a.weight_width = a.packed_width;
}

template <bool GRAD>
void launch_pack(LossArgs& a, char* ws, int64_t index, int64_t packed, hipStream_t stream) {
  a.pack_rows = (int32_t)ceil_div(max64(a.rows, 1), 512);
  const unsigned grid = (unsigned)ceil_div(max64(a.rows, 1), a.pack_rows);
  loss_pack_kernel<GRAD><<<dim3(grid + (GRAD ? 1 : 0)), dim3(256), 0, stream>>>(a, (LossMeta*)ws, (int32_t*)(ws + index),
                                                              (uint16_t*)(ws + packed));
}

template <int DT>
int run_forward(LossArgs a, const ForwardPlan& p, const Weight& w, char* ws, hipStream_t stream) {
  typedef Tiles<DT, false> T;
  launch_pack<false>(a, ws, p.index, p.packed, stream);
  for (int64_t from = 0; from < a.rows; from += p.rows_at) {
    a.row_from = (int32_t)from;
    const int64_t here = min64(p.rows_at, a.rows - from);
    a.tile_from = 0;
    for (int64_t v = 0; v < a.vocab; v += p.piece) {
      take_piece(a, w, v, p.piece, stream);
      switch (p.tile) {
        case kTile16Sum: launch_forward<typename T::T16Sum, DT>(a, here, stream); break;
        case kTile16Short: launch_forward<typename T::T16Short, DT>(a, here, stream); break;
        case kTile64Short: launch_forward<typename T::T64Short, DT>(a, here, stream); break;
        case kTile16: launch_forward<typename T::T16, DT>(a, here, stream); break;
        case kTile64: launch_forward<typename T::T64, DT>(a, here, stream); break;
        case kTileSmall: launch_forward<typename T::Small, DT>(a, here, stream); break;
        case kTile128: launch_forward<typename T::T128, DT>(a, here, stream); break;
        case kTile256: launch_forward<typename T::T256, DT>(a, here, stream); break;
      }
      a.tile_from += (int32_t)ceil_div(a.piece, logit_vocab_rows(p.tile));
    }
    if (here < 256 && !p.invariant)
      loss_join_kernel<1><<<dim3((unsigned)here), dim3(256), 0, stream>>>(a, (int32_t)p.tiles);
    else
      loss_join_kernel<16><<<dim3((unsigned)((here + 15) / 16)), dim3(256), 0, stream>>>(a, (int32_t)p.tiles);
  }
  return check_launch("cross entropy kernel");
}

template <class PZ, class PW, class PH, int DT>
void launch_piece(LossArgs a, const BackwardPlan& p, hipStream_t stream) {
  a.vocab_tiles = (int32_t)ceil_div(a.piece, PZ::MT);
  if (a.rows > 0)
    loss_dz_kernel<PZ, DT><<<dim3(grid_of(a.vocab_tiles * ceil_div(a.rows, PZ::NT))), dim3(PZ::NW * 64), 0, stream>>>(
        a, 4);
  a.vocab_tiles = (int32_t)ceil_div(a.piece, PW::NT);
  a.width_tiles = (int32_t)ceil_div(a.width, PW::MT);
  loss_dweight_kernel<PW, DT><<<dim3(grid_of(max64((int64_t)a.vocab_tiles * a.width_tiles, a.weight_sum ? p.slots : 0))),
                                dim3(PW::NW * 64), 0, stream>>>(a, 8);
  if (a.weight_sum)
    loss_dweight_sum_kernel<DT><<<dim3((unsigned)min64(a.piece, 8192)), dim3(256), 0, stream>>>(a);
  a.width_tiles = (int32_t)p.width_tiles;
  static_assert(PH::NT == PZ::NT, "one number of rows a tile");
  // at most max(slots, tiles) workgroups, whatever the count of listed rows
  if (a.rows > 0)
    loss_dhidden_product_kernel<PH, DT><<<dim3(grid_of(max64(p.width_tiles * p.row_tiles, p.slots))),
                                          dim3(PH::NW * 64), 0, stream>>>(a, 4);
}

template <int DT>
int run_backward(LossArgs a, const BackwardPlan& p, const Weight& w, char* ws, hipStream_t stream) {
  typedef Tiles<DT, false> Z;
  typedef RingProduct<DT, false, true, 2> W;  // dweight
  typedef Product<DT, 128, 128, 2, 2, 32, 2, true, true> WS;  // ... of few rows: not worth a launch that turns them
  typedef Tiles<DT, true> H;
  launch_pack<true>(a, ws, p.index, p.packed, stream);
  if (!p.few)
    loss_turn_kernel<<<dim3((unsigned)ceil_div(a.rows, 64), (unsigned)(a.packed_width / 64)), dim3(256), 0, stream>>>(
        a, (uint16_t*)(ws + p.turned));
  for (int64_t i = 0; i < p.pieces; ++i) {
    take_piece(a, w, i * p.piece, p.piece, stream);
    a.first_piece = i == 0;
    switch (p.tile) {
      case kTile16Sum: launch_piece<typename Z::T16Sum, WS, typename H::T16, DT>(a, p, stream); break;
      case kTile16Short: launch_piece<typename Z::T16Short, WS, typename H::T16, DT>(a, p, stream); break;
      case kTile64Short: launch_piece<typename Z::T64Short, WS, typename H::T64, DT>(a, p, stream); break;
      case kTile16: launch_piece<typename Z::T16, WS, typename H::T16, DT>(a, p, stream); break;
      case kTile64: launch_piece<typename Z::T64, WS, typename H::T64, DT>(a, p, stream); break;
      case kTileSmall:
        if (p.few)
          launch_piece<typename Z::Small, WS, typename H::T128, DT>(a, p, stream);
        else
          launch_piece<typename Z::Small, W, typename H::T128, DT>(a, p, stream);
        break;
      case kTile128: launch_piece<typename Z::T128, WS, typename H::T128, DT>(a, p, stream); break;
      case kTile256:
        if (p.few)
          launch_piece<typename Z::T256, WS, typename H::T256, DT>(a, p, stream);
        else
          launch_piece<typename Z::T256, W, typename H::T256, DT>(a, p, stream);
        break;
    }
  }
  if (a.sum && a.rows > 0)
    loss_dhidden_kernel<DT><<<dim3((unsigned)min64(a.rows, 4096), a.rows < 1024 ? (unsigned)ceil_div(a.width, 1024) : 1u),
                              dim3(256), 0, stream>>>(a, (int)logit_rows(p.tile));
  return check_launch("cross entropy gradient kernel");
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

// Enough for either mode: the mode may change between the query and the call.
int64_t hprms_linear_cross_entropy_workspace(int64_t rows, int64_t hidden_size, int64_t vocab, const void* weight,
                                             int64_t weight_row_stride) {
  const int rc = check_sizes(rows, hidden_size, vocab);
  if (rc != HPRMS_OK) return rc;
  const bool in_place = weight_in_place(weight, weight_row_stride, hidden_size);
  return max64(forward_plan(rows, hidden_size, vocab, in_place, false).total,
               forward_plan(rows, hidden_size, vocab, in_place, true).total);
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
  const bool in_place = weight_in_place(weight, weight_row_stride, hidden_size);
  const ForwardPlan p = forward_plan(rows, hidden_size, vocab, in_place, hprms_batch_invariant() != 0);
  rc = check_workspace(workspace, workspace_size, p.total);
  if (rc != HPRMS_OK) return rc;
  char* ws = (char*)workspace;
  LossArgs a = {};
  a.hidden = (const uint16_t*)hidden;
  a.packed = (const uint16_t*)(ws + p.packed);
  a.target = target;
  a.meta = (const LossMeta*)ws;
  a.index = (const int32_t*)(ws + p.index);
  a.hidden_stride = hidden_row_stride;
  a.packed_width = (int32_t)packed_width_of(hidden_size);
  a.ignore_index = ignore_index;
  a.rows = (int32_t)rows;
  a.width = (int32_t)hidden_size;
  a.vocab = (int32_t)vocab;
  a.loss = loss;
  a.lse = lse;
  a.target_logit = (float*)(ws + p.target_logit);
  a.partial = (float2*)(ws + p.partial);
  a.rows_at = (int32_t)p.rows_at;
  const Weight w{(const uint16_t*)weight, weight_row_stride, in_place ? nullptr : (uint16_t*)(ws + p.weight)};
  return dtype == HPRMS_DTYPE_BF16 ? run_forward<HPRMS_DTYPE_BF16>(a, p, w, ws, stream)
                                   : run_forward<HPRMS_DTYPE_FP16>(a, p, w, ws, stream);
}

int64_t hprms_linear_cross_entropy_backward_workspace(int64_t rows, int64_t hidden_size, int64_t vocab,
                                                      const void* weight, int64_t weight_row_stride) {
  const int rc = check_sizes(rows, hidden_size, vocab);
  if (rc != HPRMS_OK) return rc;
  const bool in_place = weight_in_place(weight, weight_row_stride, hidden_size);
  return max64(backward_plan(rows, hidden_size, vocab, in_place, false).total,
               backward_plan(rows, hidden_size, vocab, in_place, true).total);
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
  const bool in_place = weight_in_place(weight, weight_row_stride, hidden_size);
  const BackwardPlan p = backward_plan(rows, hidden_size, vocab, in_place, hprms_batch_invariant() != 0);
  rc = check_workspace(workspace, workspace_size, p.total);
  if (rc != HPRMS_OK) return rc;
  char* ws = (char*)workspace;
  LossArgs a = {};
  a.hidden = (const uint16_t*)hidden;
  a.packed = (const uint16_t*)(ws + p.packed);
  a.target = target;
  a.meta = (const LossMeta*)ws;
  a.index = (const int32_t*)(ws + p.index);
  a.hidden_stride = hidden_row_stride;
  a.packed_width = (int32_t)packed_width_of(hidden_size);
  a.ignore_index = ignore_index;
  a.rows = (int32_t)rows;
  a.width = (int32_t)hidden_size;
  a.vocab = (int32_t)vocab;
  a.lse = const_cast<float*>(lse);
  a.dloss = dloss;
  a.dz = (uint16_t*)(ws + p.dz);
  a.dz_stride = (int32_t)p.piece;
  a.dhidden = (uint16_t*)dhidden;
  a.dhidden_stride = dhidden_row_stride;
  a.dweight = (uint16_t*)dweight;
  a.dweight_stride = dweight_row_stride;
  a.turned = (const uint16_t*)(ws + p.turned);
  a.turned_stride = (int32_t)p.turned_stride;
  a.sum = p.shares ? (float*)(ws + p.sum) : nullptr;
  a.piece_size = (int32_t)p.piece;
  a.width_tiles = (int32_t)p.width_tiles;
  a.slots = (int32_t)p.slots;
  a.most_splits = (int32_t)p.most_splits;
  a.weight_sum = p.weight_most > 1 ? (float*)(ws + p.weight_sum) : nullptr;
  a.weight_most = (int32_t)p.weight_most;
  // without rows nothing reads the weight, which may then be null
  const Weight w{(const uint16_t*)weight, weight_row_stride,
                 in_place || rows == 0 ? nullptr : (uint16_t*)(ws + p.weight)};
  return dtype == HPRMS_DTYPE_BF16 ? run_backward<HPRMS_DTYPE_BF16>(a, p, w, ws, stream)
                                   : run_backward<HPRMS_DTYPE_FP16>(a, p, w, ws, stream);
}

}  // extern "C"
