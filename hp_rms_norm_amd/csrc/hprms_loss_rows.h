// hprms_loss_rows.h - the rows of a cross entropy call that carry a loss: the
// arguments that its kernels share, and the kernel that lists and packs those
// rows.
//
// Plain HIP without gfx950 builtins: a host build that supplies the lanes
// (threadIdx, barriers, shuffles) runs the same text.
#pragma once

#include <stdint.h>

namespace hprms {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any 2-byte boundary
typedef u32x4 u32x4_u __attribute__((aligned(2)));

// What the row list says, written by loss_pack_kernel.
struct LossMeta {
  int32_t count;   // listed rows
  float scale;     // gradient: applied to dloss
  float unscale;   // its inverse
  int32_t pad;
};

// The arguments of every loss kernel.  Listed rows are numbered by their
// position in the list ("list position").
struct LossArgs {
  const uint16_t* hidden;
  const uint16_t* weight;   // the piece's first row (the caller's, or packed)
  const int64_t* target;
  const LossMeta* meta;
  const int32_t* index;     // the row of each list position
  const uint16_t* packed;   // the listed rows' hidden values, [rows, packed_width], zeros past width
  const uint16_t* turned;   // gradient: packed transposed, [packed_width, turned_stride], zeros from count to a multiple of 64
  int64_t hidden_stride;
  int64_t ignore_index;
  int32_t weight_stride;    // elements, a multiple of 8
  int32_t weight_width;     // readable elements of a weight row, a multiple of 8
  int32_t packed_width;     // a multiple of 64
  int32_t turned_stride;    // rows rounded up to a multiple of 64
  int32_t rows;             // of the call
  int32_t width;            // elements of a hidden row
  int32_t vocab;
  int32_t piece_from, piece;  // vocabulary rows of this launch
  int32_t vocab_tiles, width_tiles;  // tiles of this launch
  // forward
  float* loss;
  float* lse;               // gradient: read
  float* target_logit;      // [rows], by list position
  float2* partial;          // [vocabulary tiles, rows_at]: maximum and sum of exponentials
  int32_t row_from, rows_at;  // list positions of this launch: [row_from, row_from + rows_at)
  int32_t tile_from;        // vocabulary tiles before this piece
  // gradient
  int32_t dz_stride;
  const float* dloss;
  uint16_t* dz;             // [rows rounded up, dz_stride], by list position
  uint16_t* dhidden;
  int64_t dhidden_stride;
  uint16_t* dweight;
  int64_t dweight_stride;
  float* sum;               // [splits, count, packed_width] shares of dhidden, by list position; null: none
  int32_t first_piece;
  int32_t piece_size, slots, most_splits;  // see splits_of
  float* weight_sum;        // [splits, piece rounded up to 128, packed_width] shares of dweight; null: none
  int32_t weight_most;      // splits of dweight at most
  int32_t pack_rows;        // rows per workgroup of the packing kernel
};

// 8 elements p[0 ... 7], of which the first n exist (n may be negative); the others read as 0
__device__ __forceinline__ u32x4 load_some(const uint16_t* p, int n) {
  if (n >= 8) return *(const u32x4_u*)p;
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) v[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
  return v;
}

// Sums over the workgroup's 256 lanes.  No wave may be reading the four words
// of lds any more; behind the call they are free again.
__device__ __forceinline__ int block_count(int v, int* lds) {
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0] + lds[1] + lds[2] + lds[3];
  __syncthreads();
  return v;
}

// The scale of dloss, by the largest of its finite magnitudes.
__device__ inline void find_scale(const LossArgs& a, LossMeta* meta, int* lds) {
  constexpr int U = 8;  // loads on their way at once
  float top = 0.0f;
  for (int32_t r = threadIdx.x; r < a.rows; r += 256 * U) {
    float g[U];
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int32_t at = min(r + u * 256, a.rows - 1);
      g[u] = fabsf(a.dloss[at]);
      t[u] = a.target[at];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g[u] < __builtin_inff() && t[u] != a.ignore_index) top = fmaxf(top, g[u]);
  }
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = __float_as_int(top);
  __syncthreads();
  for (int i = 0; i < 4; ++i) top = fmaxf(top, __int_as_float(lds[i]));
  // top = m 2^e: the scale is 2^(14 - e) / m (the exponent up to 126, so that it is finite)
  float scale = 1.0f, unscale = 1.0f;
  if (top > 0.0f) {
    const uint32_t bits = __float_as_uint(top);
    const float m = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
    const int e = max((int)(bits >> 23) - 127, -112);
    scale = ldexpf(1.0f / m, 14 - e);
    unscale = ldexpf(m, e - 14);
  }
  if (threadIdx.x == 0) {
    meta->scale = scale;
    meta->unscale = unscale;
  }
}

// Lists the rows whose target is not ignore_index, in order, and packs their
// hidden values side by side, zero up to packed_width: one operand layout for
// any width, stride and alignment, and no ignored rows in the products.  Each
// workgroup takes a.pack_rows rows, whose places it knows from counting the
// rows before them itself (at most 512 workgroups, so that those 8 bytes a row
// stay few).  The other rows get loss and lse 0, or (GRAD) a zero dhidden.
// With GRAD one workgroup more finds the scale of dloss.
template <bool GRAD>
__global__ __launch_bounds__(256) void loss_pack_kernel(LossArgs a, LossMeta* meta, int32_t* index, uint16_t* packed) {
  __shared__ int lds[4];
  __shared__ int64_t list[256];
  if constexpr (GRAD) {
    if (blockIdx.x == gridDim.x - 1) {
      find_scale(a, meta, lds);
      return;
    }
  }
  const int32_t r0 = blockIdx.x * a.pack_rows, r1 = min(r0 + a.pack_rows, a.rows);
  constexpr int U = 8;  // loads on their way at once
  // the first 256 rows' targets travel while the rows before them are counted
  int64_t target = r0 + (int)threadIdx.x < r1 ? a.target[r0 + threadIdx.x] : a.ignore_index;
  int n = 0;
  for (int32_t r = threadIdx.x; r < r0; r += 256 * U) {
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = a.target[min(r + u * 256, r0 - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) n += r + u * 256 < r0 && t[u] != a.ignore_index;
  }
  int32_t at = block_count(n, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t chunks = a.packed_width / 8;
  // up to 256 rows at a time: their places, then their 16-byte chunks in one run
  for (int32_t first = r0; first < r1; first += 256) {
    const int32_t row = first + threadIdx.x, some = min(256, r1 - first);
    const bool in = threadIdx.x < some;
    if (first > r0) target = in ? a.target[row] : a.ignore_index;
    const bool keep = in && target != a.ignore_index;
    const uint64_t mask = __ballot(keep);
    if (lane == 0) lds[wave] = __popcll(mask);
    __syncthreads();
    int before = __popcll(mask & ((uint64_t(1) << lane) - 1)), kept = 0;
    for (int i = 0; i < 4; ++i) {
      if (i < wave) before += lds[i];
      kept += lds[i];
    }
    if (keep) {
      list[before] = row;
      index[at + before] = row;
    } else if (in) {
      list[some - 1 - (threadIdx.x - before)] = row;  // the others from the end
      if constexpr (!GRAD) {
        a.loss[row] = 0.0f;
        a.lse[row] = 0.0f;
      }
    }
    __syncthreads();
    for (int32_t e = threadIdx.x; e < kept * chunks; e += 256 * U) {
      u32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int32_t x = min(e + u * 256, kept * chunks - 1), r = x / chunks, i = (x - r * chunks) * 8;
        v[u] = load_some(a.hidden + list[r] * a.hidden_stride + i, a.width - i);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)  // the listed rows lie side by side
        if (e + u * 256 < kept * chunks) *(u32x4*)(packed + (int64_t)at * a.packed_width + (e + u * 256) * 8) = v[u];
    }
    if constexpr (GRAD)
      for (int32_t r = kept; r < some; ++r)
        for (int32_t i = threadIdx.x; i < a.width; i += 256) a.dhidden[list[r] * a.dhidden_stride + i] = 0;
    at += kept;
    __syncthreads();
  }
  if (r1 == a.rows && threadIdx.x == 0) meta->count = at;
}

}  // namespace hprms
