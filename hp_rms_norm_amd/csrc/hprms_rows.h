// hprms_rows.h - what the block-edge kernels (hprms_norm_add.hip and its gradient)
// share: 16-byte row accesses at any element boundary and sums over a row's lanes.
//
// A row of H elements is H / 8 whole vectors of 8; for H % 8 != 0 the slot after
// the last whole vector holds the row's last 8 elements (H >= 8), of which only
// those that no whole vector holds count and are stored.  The others are loaded
// and set to 0 (drop_first), so it does not matter if their owner has overwritten
// them, and zeros change no sum and no maximum.  What multiplies them is either
// set to 0 as well or their product is: a weight, a gate or a reciprocal root may be
// infinite there.
#pragma once

#include <initializer_list>

#include "hprms_device.h"

namespace hprms {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// 16 and 8 bytes at any boundary (gfx950 runs global accesses unaligned)
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

__device__ __forceinline__ u32x4 load_row8(const uint16_t* p) { return *(const u32x4_any*)p; }
// of a row that is read once, past the caches if NT
template <bool NT>
__device__ __forceinline__ u32x4 load_row8_once(const uint16_t* p) {
  if constexpr (NT)
    return __builtin_nontemporal_load((const u32x4_any*)p);
  else
    return load_row8(p);
}

// Whether the rows that a call reads once are read past the caches: tensors of more
// than 2^24 elements, whose rows lie on 16-byte boundaries.  In turn over more memory
// than the caches hold 8192 x 4096 bf16 takes 45.4 us so and 47.0 through them (its
// gradient 77.4 and 82.3), 1024 x 4096 7.1 either way (22.2 and 19.9); over tensors
// that the caches still hold 42.4 and 39.1.  Off 16-byte boundaries vectors share
// lines, and 6500 x 5003 takes 57.6 and 58.7, or 56.8 and 44.0.
struct RowsRead {
  const void* base;
  int64_t stride;  // elements
};
inline bool past_caches(int64_t rows, int64_t hidden, std::initializer_list<RowsRead> read) {
  if (rows <= (int64_t(1) << 24) / hidden) return false;
  for (const RowsRead& r : read)
    if (((uintptr_t)r.base & 15) != 0 || r.stride % 8 != 0) return false;
  return true;
}

// Eight 16-bit values to p + 0 ... p + 7, without the first `skip` of them.
__device__ __forceinline__ void store_row8(uint16_t* p, u32x4 v, int skip) {
  if (skip == 0) {
    __builtin_nontemporal_store(v, (u32x4_any*)p);
  } else {
    asm volatile("" : "+v"(skip));  // or a loop's lane masks of all 7 comparisons would be kept
#pragma unroll
    for (int j = 1; j < 8; ++j)
      if (j >= skip) p[j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
  }
}

// v with its first `skip` (0 ... 7) elements 0
__device__ __forceinline__ void drop_first(u32x4& v, int skip) {
  asm volatile("" : "+v"(skip));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (skip > 2 * i) v[i] &= 0xffff0000u;
    if (skip > 2 * i + 1) v[i] = 0;
  }
}

// The same as a mask, made once for all rows of a lane.  A lane's first VPL / 2
// vectors are whole (a shape's lanes hold more than half of what they could) and need
// none.  The gradient takes masks (1021 x 5003, a gate for each element, when both were
// measured: 31.8 us, 35.5 with drop_first), the forward call, a row a workgroup, does
// not (8192 x 4096: 47.4 us with them, 46.3 without).
__device__ __forceinline__ u32x4 without_first(int skip) {
  u32x4 m;
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = skip > 2 * i + 1 ? 0u : skip > 2 * i ? 0xffff0000u : 0xffffffffu;
  return m;
}

// v through an empty asm statement: what is unpacked from it again afterwards
// need not stay in registers until then.
__device__ __forceinline__ void packed_again(u32x4& v) { asm volatile("" : "+v"(v)); }

template <int DT>
__device__ __forceinline__ float element(const u32x4& v, int j) {
  return j & 1 ? Fmt<DT>::hi(v[j / 2]) : Fmt<DT>::lo(v[j / 2]);
}

template <int DT>
__device__ __forceinline__ u32x4 pack8(const float (&o)[8]) {
  using F = Fmt<DT>;
  return u32x4{F::pack(o[0], o[1]), F::pack(o[2], o[3]), F::pack(o[4], o[5]), F::pack(o[6], o[7])};
}

// N sums over the LPR lanes of a row at once; every lane gets all of them, with
// the same bits.  `lds` holds BLOCK / 64 * N floats and is written before the one
// barrier: two calls in a row need two buffers.
template <int N, int LPR, int BLOCK>
__device__ __forceinline__ void sum_rows(float (&v)[N], float* lds) {
  constexpr int GW = LPR < 64 ? LPR : 64;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = group_sum<GW>(v[i]);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    const int wave = threadIdx.x / 64, row = threadIdx.x / LPR;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[N * wave + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[i] += lds[N * (row * W + w) + i];
    }
  }
}

// The maximum of unsigned values over the LPR lanes of a row.
template <int LPR, int BLOCK>
__device__ __forceinline__ uint32_t max_rows(uint32_t v, uint32_t* lds) {
  constexpr int GW = LPR < 64 ? LPR : 64;
  v = group_max_u32<GW>(v);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    const int wave = threadIdx.x / 64, row = threadIdx.x / LPR;
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) v = __builtin_elementwise_max(v, lds[row * W + w]);
  }
  return v;
}

}  // namespace hprms
