// hprms_int8_linear.hip - the product of 8-bit integer rows and weights with a scale
// for each row and each output feature:
//
//   out[t, o] = rne((sum_k input[t, k] * weight[o, k]) * scale[t] * weight_scale[o] + bias[o])
//
// The sums are exact in 32-bit integers (up to 131071 terms of at most 2^14), so
// their order, and with it every choice of tiles below, leaves no trace in the
// result; a sum is rounded to binary32 once (24 bits of it, a relative error of at
// most 2^-24 beside the output's own 2^-8 or 2^-11), then scaled.
//
// Few rows: the weight's bytes bound the call.  Up to 4 rows run on dot products of 4
// bytes, a wave reading whole KB of a weight's row, so the weight streams in whole
// lines (1 x 4096 x 14336: 9.9 us over three weights in turn, 10.9 over more than the
// caches hold, 5.4 TB/s; on the matrix cores 14.4; 4 x 8192 x 8192
// 15.3 and 19.6, 4 x 4096 x 4096 6.7 and 6.9, but 8 rows of it 10.1 and 6.9).  More
// rows run on the matrix cores (hprms_product.h), in tiles by a model of their
// times, and long sums of few tiles in shares.
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_product.h"

namespace hprms {
namespace {

struct Int8Args {
  const int8_t* input;
  const int8_t* weight;
  const float* scale;
  const float* weight_scale;
  const uint16_t* bias;  // null: none
  uint16_t* out;
  int64_t out_stride;
  int64_t input_stride, weight_stride;  // bytes, multiples of 16
  int32_t rows, inner, outer;           // inner: a multiple of 16
  int32_t outer_tiles, row_tiles;
  // a sum in several workgroups' shares, or null: [splits, rows, sum_stride]
  int32_t* sums;
  int32_t splits, span, sum_stride;  // span: of the summed index, a multiple of 128
};

__device__ __forceinline__ float scaled(int32_t sum, float scale, float weight_scale, float bias) {
  return __builtin_fmaf((float)sum * scale, weight_scale, bias);
}

// ---- few rows ------------------------------------------------------------------------------
__device__ __forceinline__ int32_t wave_sum(int32_t v) {
  v += (int32_t)dpp_u32<0xB1>((uint32_t)v);
  v += (int32_t)dpp_u32<0x4E>((uint32_t)v);
  v += (int32_t)dpp_u32<0x141>((uint32_t)v);
  v += (int32_t)dpp_u32<0x140>((uint32_t)v);
  v += __builtin_amdgcn_ds_swizzle(v, 0x401F);
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 32);
}

// A workgroup takes W rows of the weight and the N rows of the input; its 4 waves
// take KB of the summed index in turn.
template <int DT, int N, int W>
__global__ __launch_bounds__(256) void int8_few_rows_kernel(Int8Args a) {
  using F = Fmt<DT>;
  // KB of a row on their way at once, ahead of those in use (4 rows of 8192 x 8192:
  // 15.3 us with 1, 16.7 with 2, as fewer waves fit a CU)
  constexpr int U = N <= 2 ? 2 : 1;
  __shared__ int32_t lds[4][N * W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t first = blockIdx.x * W;
  u32x4 w[U][W], x[U][N];
  auto load = [&](int u, int32_t kb) {
    const int32_t k = kb * 1024 + lane * 16;
    const bool in = k < a.inner;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int32_t o = first + i < a.outer ? first + i : a.outer - 1;
      w[u][i] = u32x4{0, 0, 0, 0};
      if (in) w[u][i] = __builtin_nontemporal_load((const u32x4*)(a.weight + o * a.weight_stride + k));
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[u][n] = u32x4{0, 0, 0, 0};
      if (in) x[u][n] = *(const u32x4*)(a.input + n * a.input_stride + k);
    }
  };
  int32_t acc[N][W];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < W; ++i) acc[n][i] = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, wave + 4 * u);
  const int32_t kbs = (a.inner + 1023) / 1024;
  for (int32_t kb = wave; kb < kbs; kb += 4 * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[n][i] = __builtin_amdgcn_sdot4((int)x[u][n][j], (int)w[u][i][j], acc[n][i], false);
      load(u, kb + 4 * (u + U));
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int32_t s = wave_sum(acc[n][i]);
      if (lane == 0) lds[wave][n * W + i] = s;
    }
  __syncthreads();
  if (threadIdx.x >= N * W) return;
  const int32_t t = threadIdx.x / W, o = first + threadIdx.x % W;
  if (o >= a.outer) return;
  const int32_t s = lds[0][threadIdx.x] + lds[1][threadIdx.x] + lds[2][threadIdx.x] + lds[3][threadIdx.x];
  const float bias = a.bias ? F::one(a.bias[o]) : 0.0f;
  a.out[t * a.out_stride + o] = F::pack1(scaled(s, a.scale[t], a.weight_scale[o], bias));
}

// ---- tiles on the matrix cores ---------------------------------------------------------------
// A: the weight's rows, so that a lane's four sums are neighbours of an output row.
template <class P>
constexpr int kLdsBytes = P::LDS_BYTES > kTileOutBytes<P> ? P::LDS_BYTES : kTileOutBytes<P>;

template <class P, int DT>
__global__ __launch_bounds__(P::NW * 64) void int8_tile_kernel(Int8Args a, int group) {
  using F = Fmt<DT>;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[kLdsBytes<P> / 2];
  int m, ns;
  if (!tile_of(blockIdx.x, a.outer_tiles, a.row_tiles * a.splits, group, &m, &ns)) return;
  const int n = ns % a.row_tiles, split = ns / a.row_tiles, from = split * a.span;
  const int m0 = m * P::MT, n0 = n * P::NT;
  const int depth = a.inner - from < a.span ? a.inner - from : a.span;
  const Operand weight = {(const uint16_t*)(a.weight + m0 * a.weight_stride + from),
                          (a.outer - 1 - m0) * a.weight_stride + a.inner - from, (int32_t)(a.weight_stride / 2)};
  const Operand input = {(const uint16_t*)(a.input + n0 * a.input_stride + from),
                         (a.rows - 1 - n0) * a.input_stride + a.inner - from, (int32_t)(a.input_stride / 2)};
  f32x4 acc[P::MI][P::NI];
  P::run(weight, input, depth / 2, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::WN % P::WM, wn = wave % P::WN;
  const bool one = P::NW > P::WM * P::WN;  // a SumProduct's waves all hold the tile: the first writes it
  if (one && wave > 0) return;
  if (a.sums) {
    int32_t* to = a.sums + (int64_t)split * a.rows * a.sum_stride;
#pragma unroll
    for (int ni = 0; ni < P::NI; ++ni) {
      const int t = n0 + (wn * P::NI + ni) * 16 + (lane & 15);
      if (t >= a.rows) continue;
#pragma unroll
      for (int mi = 0; mi < P::MI; ++mi) {
        const int o = m0 + (wm * P::MI + mi) * 16 + (lane >> 4) * 4;
        if (o < a.outer) *(f32x4*)(to + (int64_t)t * a.sum_stride + o) = acc[mi][ni];
      }
    }
    return;
  }
  float scale[P::NI];
#pragma unroll
  for (int ni = 0; ni < P::NI; ++ni) {
    const int t = n0 + (wn * P::NI + ni) * 16 + (lane & 15);
    scale[ni] = t < a.rows ? a.scale[t] : 0.0f;
  }
  // the features' scales and biases, read once for all rows of the tile
  typedef f32x4 f32x4_any __attribute__((aligned(4)));
  f32x4 weight_scale[P::MI];
  u32x2 bias[P::MI];
#pragma unroll
  for (int mi = 0; mi < P::MI; ++mi) {
    const int o = m0 + (wm * P::MI + mi) * 16 + (lane >> 4) * 4;
    bias[mi] = u32x2{0, 0};
    if (o + 4 <= a.outer) {
      weight_scale[mi] = *(const f32x4_any*)(a.weight_scale + o);
      if (a.bias) bias[mi] = *(const u32x2_out*)(a.bias + o);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = o + i < a.outer ? o + i : a.outer - 1;
        weight_scale[mi][i] = a.weight_scale[at];
        if (a.bias) bias[mi][i / 2] |= (uint32_t)a.bias[at] << (16 * (i & 1));
      }
    }
  }
  // a fragment's four values
  auto value = [&](int mi, int ni) {
    const i32x4 s = __builtin_bit_cast(i32x4, acc[mi][ni]);
    float d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d[i] = scaled(s[i], scale[ni], weight_scale[mi][i], i & 1 ? F::hi(bias[mi][i / 2]) : F::lo(bias[mi][i / 2]));
    return u32x2{F::pack(d[0], d[1]), F::pack(d[2], d[3])};
  };
  if constexpr (P::NW > P::WM * P::WN) {
#pragma unroll
    for (int ni = 0; ni < P::NI; ++ni) {
      const int t = n0 + ni * 16 + (lane & 15);
      if (t >= a.rows) continue;
#pragma unroll
      for (int mi = 0; mi < P::MI; ++mi) {
        const int o = m0 + mi * 16 + (lane >> 4) * 4;
        const u32x2 v = value(mi, ni);
        for (int i = 0; i < 4 && o + i < a.outer; ++i)
          a.out[t * a.out_stride + o + i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
      }
    }
  } else {
    tile_out<P>(lds, a.outer - m0, value,
                [&](int row) { return n0 + row < a.rows ? a.out + (n0 + row) * a.out_stride + m0 : nullptr; });
  }
}

// The output from its sums' shares, four neighbours a lane.
template <int DT>
__global__ __launch_bounds__(256) void int8_sum_kernel(Int8Args a) {
  using F = Fmt<DT>;
  const int o = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (o >= a.outer) return;
  for (int t = blockIdx.y; t < a.rows; t += gridDim.y) {
    const int32_t* from = a.sums + (int64_t)t * a.sum_stride + o;
    i32x4 s = {0, 0, 0, 0};
    constexpr int U = 8;  // loads on their way at once
    for (int i = 0; i < a.splits; i += U) {
      i32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = i + u < a.splits ? *(const i32x4*)(from + (int64_t)(i + u) * a.rows * a.sum_stride) : i32x4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u];
    }
    const float scale = a.scale[t];
    uint16_t* to = a.out + t * a.out_stride + o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (o + i < a.outer)
        to[i] = F::pack1(scaled(s[i], scale, a.weight_scale[o + i], a.bias ? F::one(a.bias[o + i]) : 0.0f));
  }
}

// Rows that 16-byte loads at 16-byte boundaries cannot take in place, copied to
// rows of whole 16 bytes with zeros behind: 16 bytes a lane, of the input's rows,
// then of the weight's.
struct PackJob {
  const int8_t* from;
  int8_t* to;
  int64_t stride, chunks;  // chunks: rows x 16-byte pieces, 0 for none
};

__global__ __launch_bounds__(256) void int8_pack_kernel(PackJob input, PackJob weight, int32_t width,
                                                        int32_t row_chunks) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < input.chunks + weight.chunks; at += step) {
    const bool second = at >= input.chunks;
    const PackJob& job = second ? weight : input;
    const int64_t c = second ? at - input.chunks : at;
    const int64_t row = (c | row_chunks) >> 31 ? c / row_chunks : (int64_t)((uint32_t)c / (uint32_t)row_chunks);
    const int32_t k = (int32_t)(c - row * row_chunks) * 16;
    const int8_t* f = job.from + row * job.stride + k;
    u32x4 v = {0, 0, 0, 0};
    if (k + 16 <= width) {
      typedef u32x4 u32x4_any __attribute__((aligned(1)));
      v = *(const u32x4_any*)f;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k + j < width) v[j / 4] |= (uint32_t)(uint8_t)f[j] << (8 * (j & 3));
    }
    *(u32x4*)(job.to + c * 16) = v;
  }
}

// ---- host ------------------------------------------------------------------------------
constexpr int64_t kMaxInner = 131071;  // 2^14 each, below 2^31 together
// a tile's 256 rows at this stride stay within a buffer access's 31-bit offset
constexpr int64_t kMaxStride = int64_t(1) << 22;

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t ceil_div(int64_t v, int64_t m) { return (v + m - 1) / m; }
bool aligned_to(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

bool in_place(const void* p, int64_t stride, int64_t inner) {
  return aligned_to(p, 16) && stride % 16 == 0 && inner % 16 == 0 && stride <= kMaxStride;
}

// Tiles of output features x rows, and what a workgroup of them takes for 128
// summed entries, ns, with `round` workgroups on 256 CUs at once, or `alone` with
// one a CU at most (a slice's latency).  Measured at 4 to 1024 rows of 4096 to 4096,
// 4096 to 14336, 14336 to 4096 and 4096 to 1024, where a call takes 2.5 us besides.
// The model's choice is the fastest of these, or within 13% of it, at all of them,
// e.g. (us; model's first) 48 x 4096 x 4096 64 x 16 8.4, 64 x 32 10.9, 64 x 64 14.0; 24 x
// 4096 x 14336 64 x 32 14.4, 64 x 16 16.7; 512 x 4096 x 14336 128 x 128 41.6, 256 x
// 256 48.5, 64 x 128 56; 1024 x 4096 x 14336 256 x 256 53.6, 128 x 128 81; 256 x 4096 x
// 14336 64 x 128 32.2, 128 x 128 40.8.  The two smallest take slices of 256 bytes in
// 3 stages: 48 x 4096 x 4096 8.4 us, with 128 bytes in 6 stages, twice the barriers,
// 10.6 (64 x 64 so: 128 x 4096 x 14336 26.5, one workgroup a CU, as it is 20 to 23).
enum Tile { kFewRows, kSum16, k64x16, k64x32, k64x64, k64x128, k128x128, k256x256 };
struct TileCost {
  Tile tile;
  int32_t outer, rows, round, ns, alone;
};
constexpr TileCost kTiles[] = {{kSum16, 16, 16, 256, 140, 140},       {k64x16, 64, 16, 512, 300, 190},
                               {k64x32, 64, 32, 512, 480, 275},       {k64x64, 64, 64, 512, 550, 470},
                               {k64x128, 64, 128, 512, 900, 765},     {k128x128, 128, 128, 512, 1300, 1105},
                               {k256x256, 256, 256, 256, 1660, 1660}};
constexpr int64_t kSplitInner = 8192, kLeastShare = 1792;

struct Choice {
  Tile tile;
  int32_t splits, span;
};

// A sum of 8192 entries or more is cut into shares, of 1792 at least, where that
// fills the CUs: a second launch, 3 us, adds them (4 bytes of each written and read
// again).  Whole and in shares, us: 16 x 14336 x 4096 18.5 and 15.7, 48 rows 27.0 and
// 18.8, 256 rows 39.3 and 35.3; 24 x 16384 x 4096 29.7 and 18.8; 24 x 8192 x 1024
// 10.6 and 8.4.  With many outputs the model takes shares where the whole sum is
// faster: 16 x 8192 x 8192 18.5 and 17.9, but 48 rows 19.6 and 21.0, 128 rows 25.0 and
// 30.7.  At 4096 entries they gain nothing (48 x 4096 x 4096 8.2 either way, x 14336
// 16.1 and 18.3).
Choice choose(int64_t rows, int64_t inner, int64_t outer) {
  if (rows <= 4) return {kFewRows, 1, (int32_t)inner};
  Choice best = {};
  double least = 0.0;
  for (const TileCost& t : kTiles) {
    const int64_t tiles = ceil_div(outer, t.outer) * ceil_div(rows, t.rows);
    const double round = (double)t.round * current_cus() / kRefCUs;
    int64_t most = inner >= kSplitInner && t.tile != kSum16 ? inner / kLeastShare : 1;
    for (int64_t splits = 1; splits <= most; splits *= 2) {
      if (splits > 1 && (double)(tiles * splits) > round) break;
      const int64_t span = round_up(ceil_div(inner, splits), 128);
      double us = (double)ceil_div(span, 128) * 1e-3 *
                  (tiles * splits <= current_cus() ? t.alone : t.ns * (double)ceil_div(tiles * splits, (int64_t)round));
      if (splits > 1) us += 3.0 + (double)rows * outer * splits * 8 / 5e6;
      if (best.tile == kFewRows || us < least) {
        best = {t.tile, (int32_t)ceil_div(inner, span), (int32_t)span};
        least = us;
      }
    }
  }
  return best;
}

struct Plan {
  int64_t packed_inner, weight, sums, total;  // bytes; the packed input at 0
  bool input_in_place, weight_in_place;
  Choice choice;
};
Plan plan_of(int64_t rows, int64_t inner, int64_t outer, const void* input, int64_t input_stride, const void* weight,
             int64_t weight_stride) {
  Plan p;
  p.packed_inner = round_up(inner, 16);
  p.input_in_place = in_place(input, input_stride, inner);
  p.weight_in_place = in_place(weight, weight_stride, inner);
  p.choice = choose(rows, p.packed_inner, outer);
  p.weight = p.input_in_place ? 0 : round_up(rows * p.packed_inner, 256);
  p.sums = p.weight + (p.weight_in_place ? 0 : round_up(outer * p.packed_inner, 256));
  p.total = p.sums + (p.choice.splits > 1 ? p.choice.splits * rows * round_up(outer, 4) * 4 : 0);
  return p;
}

int check_sizes(int64_t rows, int64_t inner, int64_t outer) {
  if (rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)rows);
  if (inner < 1 || outer < 1)
    return fail(HPRMS_E_INVALID, "inner and outer must be >= 1 (got %lld, %lld)", (long long)inner, (long long)outer);
  if (inner > kMaxInner)
    return fail(HPRMS_E_RANGE, "inner %lld exceeds %lld: its sums would not fit 32 bits", (long long)inner,
                (long long)kMaxInner);
  if (rows > int64_t(1) << 24 || outer > int64_t(1) << 24)
    return fail(HPRMS_E_RANGE, "rows and outer must be at most 2^24 (got %lld, %lld)", (long long)rows,
                (long long)outer);
  if (ceil_div(rows, 128) * ceil_div(outer, 128) > int64_t(1) << 22)  // a launch holds fewer than 2^32 work-items
    return fail(HPRMS_E_RANGE, "the output holds more than 2^36 elements (%lld x %lld)", (long long)rows,
                (long long)outer);
  return HPRMS_OK;
}

template <class P, int DT>
void launch_tiles(Int8Args a, hipStream_t stream) {
  a.outer_tiles = (int32_t)ceil_div(a.outer, P::MT);
  a.row_tiles = (int32_t)ceil_div(a.rows, P::NT);
  const int64_t tiles = (int64_t)a.outer_tiles * a.row_tiles * a.splits;
  int8_tile_kernel<P, DT><<<dim3((unsigned)round_up(tiles, 8)), dim3(P::NW * 64), 0, stream>>>(a, 8);
  if (a.sums)
    int8_sum_kernel<DT><<<dim3((unsigned)ceil_div(a.outer, 1024), (unsigned)(a.rows < 8192 ? a.rows : 8192)),
                          dim3(256), 0, stream>>>(a);
}

template <int DT, int N, int W>
void launch_few(const Int8Args& a, hipStream_t stream) {
  int8_few_rows_kernel<DT, N, W><<<dim3((unsigned)ceil_div(a.outer, W)), dim3(256), 0, stream>>>(a);
}

template <int DT>
int launch_all(const Int8Args& a, Tile tile, hipStream_t stream) {
  constexpr int I = kInt8Pairs;
  switch (tile) {
    case kFewRows:
      if (a.rows == 1)
        launch_few<DT, 1, 4>(a, stream);
      else if (a.rows == 2)
        launch_few<DT, 2, 4>(a, stream);
      else if (a.rows == 3)
        launch_few<DT, 3, 4>(a, stream);
      else
        launch_few<DT, 4, 4>(a, stream);
      break;
    case kSum16: launch_tiles<SumProduct<I, 1, 1, 8, 4>, DT>(a, stream); break;
    case k64x16: launch_tiles<Product<I, 64, 16, 4, 1, 128, 3, false, false>, DT>(a, stream); break;
    case k64x32: launch_tiles<Product<I, 64, 32, 4, 1, 128, 3, false, false>, DT>(a, stream); break;
    case k64x64: launch_tiles<Product<I, 64, 64, 2, 2, 64, 4, false, false>, DT>(a, stream); break;
    case k64x128: launch_tiles<Product<I, 64, 128, 2, 2, 64, 3, false, false>, DT>(a, stream); break;
    case k128x128: launch_tiles<Product<I, 128, 128, 2, 2, 64, 2, false, false>, DT>(a, stream); break;
    case k256x256: launch_tiles<RingProduct<I, false, false, 2>, DT>(a, stream); break;
  }
  return check_launch("8-bit linear kernel");
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_int8_linear_workspace(int64_t rows, int64_t inner, int64_t outer, const void* input,
                                    int64_t input_row_stride, const void* weight, int64_t weight_row_stride) {
  const int rc = check_sizes(rows, inner, outer);
  return rc != HPRMS_OK ? rc : rows == 0 ? 0
                                         : plan_of(rows, inner, outer, input, input_row_stride, weight,
                                                   weight_row_stride)
                                               .total;
}

int hprms_int8_linear(void* out, const void* input, const float* scale, const void* weight, const float* weight_scale,
                      const void* bias, void* workspace, int64_t workspace_size, int64_t rows, int64_t inner,
                      int64_t outer, int64_t out_row_stride, int64_t input_row_stride, int64_t weight_row_stride,
                      int dtype, hipStream_t stream) {
  if (dtype != HPRMS_DTYPE_BF16 && dtype != HPRMS_DTYPE_FP16)
    return fail(HPRMS_E_INVALID, "dtype must be HPRMS_DTYPE_BF16 or HPRMS_DTYPE_FP16 (got %d)", dtype);
  const int rc = check_sizes(rows, inner, outer);
  if (rc != HPRMS_OK) return rc;
  if (out_row_stride < outer || input_row_stride < inner || weight_row_stride < inner)
    return fail(HPRMS_E_INVALID, "row strides must be >= the rows' widths");
  if (!extent_ok(rows, out_row_stride, 2, outer) || !extent_ok(rows, input_row_stride, 1, inner) ||
      !extent_ok(outer, weight_row_stride, 1, inner))
    return fail(HPRMS_E_RANGE, "the rows at these row strides span more than 2^56 bytes");
  if (rows == 0) return HPRMS_OK;
  if (!out || !input || !scale || !weight || !weight_scale) return fail(HPRMS_E_INVALID, "null tensor pointer");
  if (!aligned_to(out, 2) || !aligned_to(scale, 4) || !aligned_to(weight_scale, 4) || !aligned_to(bias, 2))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  const Plan p = plan_of(rows, inner, outer, input, input_row_stride, weight, weight_row_stride);
  if (p.total > 0 && (!workspace || workspace_size < p.total || !aligned_to(workspace, 256)))
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 256-byte aligned (got %lld)", (long long)p.total,
                (long long)workspace_size);
  char* ws = (char*)workspace;
  Int8Args a = {};
  a.input = (const int8_t*)input;
  a.input_stride = input_row_stride;
  a.weight = (const int8_t*)weight;
  a.weight_stride = weight_row_stride;
  PackJob jobs[2] = {};
  if (!p.input_in_place) {
    jobs[0] = {a.input, (int8_t*)ws, a.input_stride, rows * (p.packed_inner / 16)};
    a.input = (const int8_t*)ws;
    a.input_stride = p.packed_inner;
  }
  if (!p.weight_in_place) {
    jobs[1] = {a.weight, (int8_t*)(ws + p.weight), a.weight_stride, outer * (p.packed_inner / 16)};
    a.weight = (const int8_t*)(ws + p.weight);
    a.weight_stride = p.packed_inner;
  }
  if (const int64_t chunks = jobs[0].chunks + jobs[1].chunks) {
    const int64_t groups = ceil_div(chunks, 256);
    int8_pack_kernel<<<dim3((unsigned)(groups < 16384 ? groups : 16384)), dim3(256), 0, stream>>>(
        jobs[0], jobs[1], (int32_t)inner, (int32_t)(p.packed_inner / 16));
  }
  a.scale = scale;
  a.weight_scale = weight_scale;
  a.bias = (const uint16_t*)bias;
  a.out = (uint16_t*)out;
  a.out_stride = out_row_stride;
  a.rows = (int32_t)rows;
  a.inner = (int32_t)p.packed_inner;
  a.splits = p.choice.splits;
  a.span = p.choice.span;
  a.sum_stride = (int32_t)round_up(outer, 4);
  if (a.splits > 1) a.sums = (int32_t*)(ws + p.sums);
  a.outer = (int32_t)outer;
  return dtype == HPRMS_DTYPE_BF16 ? launch_all<HPRMS_DTYPE_BF16>(a, p.choice.tile, stream)
                                   : launch_all<HPRMS_DTYPE_FP16>(a, p.choice.tile, stream);
}

}  // extern "C"
