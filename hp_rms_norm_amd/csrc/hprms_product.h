// hprms_product.h - the tile product of the loss and of the 8-bit linear kernels: C
// = A . B^T on the matrix cores, over 16-bit operands with binary32 sums or over
// 8-bit integers with 32-bit integer sums.
#pragma once

#include "hprms_device.h"

namespace hprms {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
// 16 and 8 bytes at any 2-byte boundary
typedef u32x4 u32x4_out __attribute__((aligned(2)));
typedef u32x2 u32x2_out __attribute__((aligned(2)));

// 8-bit integers as a product's element type: everything below counts in pairs of
// them, 16 bits each, and an accumulator's registers hold integers.  (A lane of
// v_mfma_i32_16x16x64_i8 holds 16 bytes of a row at byte 16 (l / 16), as one of
// v_mfma_f32_16x16x32 does.)  Pairs cannot lie k outer.
constexpr int kInt8Pairs = 16;

template <int DT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == kInt8Pairs)
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                                                           __builtin_bit_cast(i32x4, b),
                                                                           __builtin_bit_cast(i32x4, c), 0, 0, 0));
  else if constexpr (DT == HPRMS_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <int DT>
__device__ __forceinline__ f32x4 add_sums(f32x4 a, f32x4 b) {
  if constexpr (DT == kInt8Pairs)
    return __builtin_bit_cast(f32x4, __builtin_bit_cast(i32x4, a) + __builtin_bit_cast(i32x4, b));
  else
    return a + b;
}

// One operand of a tile: `rows` of its first index (the tile's extent) over the
// summed index k.
//   KOUTER false: element (r, k) at base + r * stride + k (k contiguous)
//   KOUTER true:  element (r, k) at base + k * stride + r (r contiguous)
// `bytes` from base hold the operand: what lies past them reads as 0.
struct Operand {
  const uint16_t* base;
  int64_t bytes;
  int32_t stride;  // elements, a multiple of 8
};

typedef __attribute__((address_space(3))) uint16_t lds_u16;

// vmcnt(vm) lgkmcnt(0): all but the last vm loads and every LDS read are done
constexpr int wait_code(int vm) { return (vm & 15) | (vm >> 4) << 14 | 0x70; }

// The workgroup's barrier, which neither memory accesses nor products pass.
__device__ __forceinline__ void phase_end() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// A workgroup of WM x WN waves computes an MT x NT tile, each wave MI x NI
// fragments of 16 x 16.  Slices of BK summed entries travel from memory to LDS
// without registers (16 bytes a lane), ST slices deep; a slice's LDS rows are
// swizzled through the addresses that the lanes load from, so that fragment
// reads touch every bank once:
//   k contiguous: LDS row r holds 2 * BK bytes, its 16-byte chunk p the row's
//     chunk p ^ (r mod 16) (BK = 128), p ^ (r mod 8) (64) or p ^ (r / 2 mod 4) (32); a
//     fragment is one 16-byte read a lane.
//   k outer: LDS row k holds 2 * extent bytes, its 32-byte unit u the unit
//     u ^ (k mod 4 + 4 (k / 8 mod 2)), as far as the extent has units; a
//     fragment is two transposing 8-byte reads a lane, which give each 16 lanes
//     4 entries of 16 columns.
//
// With 8 waves the two halves of the workgroup run one phase apart, as in
// RingProduct below (256 x 128 x 4096 tiles, two workgroups a CU: 999 TFLOP/s
// against 985 without).
template <int DT, int MT_, int NT_, int WM_, int WN_, int BK_, int ST_, bool AKO_, bool BKO_>
struct Product {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, BK = BK_, ST = ST_;
  static constexpr bool AKO = AKO_, BKO = BKO_;
  static constexpr int NW = WM * WN;
  static constexpr int MI = MT / WM / 16, NI = NT / WN / 16;
  static constexpr int ABYTES = MT * BK * 2, BBYTES = NT * BK * 2;
  static constexpr int STAGE = ABYTES + BBYTES;
  static constexpr int LA = (ABYTES / 1024 + NW - 1) / NW, LB = (BBYTES / 1024 + NW - 1) / NW;
  static constexpr int LDS_BYTES = STAGE * ST;
  static_assert(BK == 128 || BK == 64 || BK == 32, "slice depth");
  static_assert(MT % (WM * 16) == 0 && NT % (WN * 16) == 0, "wave tiles");
  static_assert(ABYTES % 1024 == 0 && BBYTES % 1024 == 0, "whole loads");

  // What a row's 16-byte chunks are permuted by (k contiguous).
  __device__ static __forceinline__ int swizzle(int r) { return BK == 128 ? r & 15 : BK == 64 ? r & 7 : (r >> 1) & 3; }

  // Byte offset, from the operand's base, of what lane `lane` loads in load j
  // of a slice (1024 bytes of LDS), for an operand of EXT rows; *k: the slice's
  // summed entry where the lane's 8 elements begin (k contiguous).
  template <int EXT, bool KO>
  __device__ static __forceinline__ uint32_t load_offset(int j, int lane, int32_t stride, int* k) {
    const int at = j * 1024 + lane * 16;  // byte in the slice
    if constexpr (!KO) {
      constexpr int RB = BK * 2;
      const int r = at / RB, p = at % RB / 16;
      const int c = p ^ swizzle(r);
      *k = c * 8;
      return ((uint32_t)r * (uint32_t)stride + c * 8) * 2;
    } else {
      constexpr int RB = EXT * 2;
      const int kr = at / RB, p = at % RB / 16;
      const int u = (p >> 1) ^ swizzle_k<EXT>(kr);
      *k = 0;
      return ((uint32_t)kr * (uint32_t)stride + u * 16 + (p & 1) * 8) * 2;
    }
  }
  template <int EXT>
  __device__ static __forceinline__ int swizzle_k(int k) {
    constexpr int UNITS = EXT / 16;
    return ((k & 3) | (k >> 1 & 4)) & (UNITS - 1 < 7 ? UNITS - 1 : 7);
  }

  // The fragment of rows r0 ... r0 + 15 and entries kk * 32 ... + 31 of a slice.
  template <int EXT, bool KO>
  __device__ static __forceinline__ u32x4 fragment(lds_u16* slice, int r0, int kk, int lane) {
    if constexpr (!KO) {
      const int r = r0 + (lane & 15), c = kk * 4 + (lane >> 4);
      const int p = c ^ swizzle(r);
      return *(__attribute__((address_space(3))) u32x4*)(slice + r * BK + p * 8);
    } else {
      // 16 lanes read 4 rows of k (lane & 15) / 4, 4 columns each
      const int k = kk * 32 + (lane >> 4) * 8 + ((lane & 15) >> 2);
      const int u = (r0 / 16) ^ swizzle_k<EXT>(k);
      lds_u16* p = slice + k * EXT + u * 16 + (lane & 3) * 4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      const s16x4 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * EXT));
      const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
      return u32x4{l[0], l[1], h[0], h[1]};
    }
  }

  // Behind it every wave's share of the oldest of the ST - 1 slices on their
  // way is in LDS, and every fragment read before it in registers.
  __device__ static __forceinline__ void landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_code((ST - 2) * (LA + LB)));
    phase_end();
  }

  // acc <- A . B^T over k in [0, depth).
  __device__ static __forceinline__ void run(const Operand& a, const Operand& b, int32_t depth, uint16_t* lds_generic,
                                             f32x4 (&acc)[MI][NI]) {
    lds_u16* lds = (lds_u16*)lds_generic;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    uint32_t oa[LA], ob[LB];
    int ka[LA], kb[LB];
    int ja[LA], jb[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      // waves without a load of their own repeat the last one
      ja[i] = i * NW + wave < ABYTES / 1024 ? i * NW + wave : ABYTES / 1024 - 1;
      oa[i] = load_offset<MT, AKO>(ja[i], lane, a.stride, &ka[i]);
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      jb[i] = i * NW + wave < BBYTES / 1024 ? i * NW + wave : BBYTES / 1024 - 1;
      ob[i] = load_offset<NT, BKO>(jb[i], lane, b.stride, &kb[i]);
    }
    const int32_t slices = (depth + BK - 1) / BK;
    const int64_t astep = AKO ? (int64_t)a.stride * BK * 2 : BK * 2;
    const int64_t bstep = BKO ? (int64_t)b.stride * BK * 2 : BK * 2;
    const char* abase = (const char*)a.base;
    const char* bbase = (const char*)b.base;
    int64_t abytes = a.bytes, bbytes = b.bytes;

    // loads of slice t into LDS stage s; past the last slice nothing is in range
    auto load = [&](int32_t t, int s) {
      const bool in = t < slices;
      const int64_t an = !in || abytes < 0 ? 0 : abytes > 0x7fffffff ? 0x7fffffff : abytes;
      const int64_t bn = !in || bbytes < 0 ? 0 : bbytes > 0x7fffffff ? 0x7fffffff : bbytes;
      const __amdgpu_buffer_rsrc_t ra = make_rsrc(abase, (uint32_t)an);
      const __amdgpu_buffer_rsrc_t rb = make_rsrc(bbase, (uint32_t)bn);
      lds_u16* stage = lds + s * (STAGE / 2);
      const int left = depth - t * BK;  // entries of k from this slice on
#pragma unroll
      for (int i = 0; i < LA; ++i) {
        const uint32_t off = !AKO && ka[i] >= left ? kOOB : oa[i];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(stage + ja[i] * 512), 16,
                                                 off, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < LB; ++i) {
        const uint32_t off = !BKO && kb[i] >= left ? kOOB : ob[i];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rb, (__attribute__((address_space(3))) void*)(stage + ABYTES / 2 + jb[i] * 512), 16, off, 0, 0, 0);
      }
      abase += astep;
      abytes -= astep;
      bbase += bstep;
      bbytes -= bstep;
    };

#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) load(s, s);
    int s = 0;
    if constexpr (NW == 8) {
      static_assert(BK == 32, "one step of 32 entries a phase");
      const bool late = wave >= NW / 2;
      landed();
      if (late) phase_end();
      for (int32_t t = 0; t < slices; ++t) {
        lds_u16* as = lds + s * (STAGE / 2);
        lds_u16* bs = as + ABYTES / 2;
        u32x4 fa[MI], fb[NI];
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[j] = fragment<NT, BKO>(bs, (wn * NI + j) * 16, 0, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[i] = fragment<MT, AKO>(as, (wm * MI + i) * 16, 0, lane);
        __builtin_amdgcn_sched_barrier(0);
        // into the stage of slice t - 1, which the other half read in the last phase
        load(t + ST - 1, s == 0 ? ST - 1 : s - 1);
        landed();  // slice t + 1, which the other half reads (or has begun to) from the next phase on
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = mfma16<DT>(fa[i], fb[j], acc[i][j]);
        __builtin_amdgcn_s_setprio(0);
        phase_end();
        s = s + 1 == ST ? 0 : s + 1;
      }
      if (!late) phase_end();
    } else {
      for (int32_t t = 0; t < slices; ++t) {
        landed();
        load(t + ST - 1, s == 0 ? ST - 1 : s - 1);
        lds_u16* as = lds + s * (STAGE / 2);
        lds_u16* bs = as + ABYTES / 2;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
          u32x4 fa[MI], fb[NI];
#pragma unroll
          for (int i = 0; i < MI; ++i) fa[i] = fragment<MT, AKO>(as, (wm * MI + i) * 16, kk, lane);
#pragma unroll
          for (int j = 0; j < NI; ++j) fb[j] = fragment<NT, BKO>(bs, (wn * NI + j) * 16, kk, lane);
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma16<DT>(fa[i], fb[j], acc[i][j]);
        }
        s = s + 1 == ST ? 0 : s + 1;
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_code(0));  // LDS is free again behind the next barrier
  }
};

// Few tiles over a long sum: the waves of a workgroup share one tile of MI x NI
// fragments and take the summed entries in turn, 64 at a time, from memory
// straight to registers, D of their turns ahead; both operands k contiguous.  The
// waves' sums are joined through LDS in a fixed order, and every wave holds the
// whole tile afterwards (WM = WN = 1).  A tile's time is its latency: a slice of
// Product above costs a workgroup that is alone on its CU 0.3 us, its barrier
// and its way through LDS, however many slices are on their way (71 slices: 21
// us with 6 or 15 stages), while here 4 waves go through them at 9.0 us.  With
// many tiles loads of half lines tell (16 rows of 60000 x 4096: 3.7 TB/s, 6 there).
template <int DT, int MI_, int NI_, int NW_, int D>
struct SumProduct {
  static constexpr int MI = MI_, NI = NI_, MT = MI * 16, NT = NI * 16, NW = NW_, WM = 1, WN = 1;
  static constexpr int LDS_BYTES = NW * MI * NI * 1024;

  __device__ static __forceinline__ void run(const Operand& a, const Operand& b, int32_t depth, uint16_t* lds_generic,
                                             f32x4 (&acc)[MI][NI]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, k0 = (lane >> 4) * 8;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(a.base, a.bytes < 0x7fffffff ? (uint32_t)a.bytes : 0x7fffffffu);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(b.base, b.bytes < 0x7fffffff ? (uint32_t)b.bytes : 0x7fffffffu);
    uint32_t oa[MI], ob[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) oa[i] = ((uint32_t)(i * 16 + r) * (uint32_t)a.stride + k0) * 2;
#pragma unroll
    for (int j = 0; j < NI; ++j) ob[j] = ((uint32_t)(j * 16 + r) * (uint32_t)b.stride + k0) * 2;
    u32x4 fa[D][2][MI], fb[D][2][NI];
    // the two steps of slice t; past the depth nothing is in range
    auto load = [&](int t, u32x4 (&va)[2][MI], u32x4 (&vb)[2][NI]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = t * 64 + h * 32;
        const bool in = k + k0 < depth;
#pragma unroll
        for (int i = 0; i < MI; ++i)
          va[h][i] = __builtin_amdgcn_raw_buffer_load_b128(ra, in ? oa[i] + k * 2 : kOOB, 0, 0);
#pragma unroll
        for (int j = 0; j < NI; ++j)
          vb[h][j] = __builtin_amdgcn_raw_buffer_load_b128(rb, in ? ob[j] + k * 2 : kOOB, 0, 0);
      }
    };
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < D; ++d) load(wave + d * NW, fa[d], fb[d]);
    const int32_t slices = (depth + 63) / 64;
    for (int32_t t = wave; t < slices; t += D * NW) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma16<DT>(fa[d][h][i], fb[d][h][j], acc[i][j]);
        load(t + (d + D) * NW, fa[d], fb[d]);
      }
    }
    f32x4* lds = (f32x4*)lds_generic;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) lds[((wave * MI + i) * NI + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        acc[i][j] = lds[(i * NI + j) * 64 + lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) acc[i][j] = add_sums<DT>(acc[i][j], lds[((w * MI + i) * NI + j) * 64 + lane]);
      }
  }
};

// The 256 x 256 tile of 8 waves: WM x 8 / WM, 64 x 128 or 128 x 64 each.
//
// LDS holds 10 chunks of 16 KB.  A slice of 64 summed entries is 4 of them, two
// of A and two of B: 128 rows of 64 entries each (k contiguous) or all 256
// rows' 32 entries (k outer), so that a load instruction takes whole 128-byte
// lines (8 rows of 128 bytes, or 2 of 512).  Chunk c of the product lies at
// place c mod 10: while slice t is in use, the four places that slice t - 1
// left take B of slice t + 1 and A of slice t + 2.
//
// The waves of the second half (w + 4 shares a SIMD with w) run one phase
// behind those of the first; the workgroup's barrier ends every phase, and a
// phase is either the fragment reads of half a slice and 4 loads, or that
// half's products, so each SIMD's matrix core works for one wave while the
// other's fragments arrive.  Without that both waves of a SIMD wait for LDS at
// the same time.
//
// 1.1 TFLOP of each kind, tiles in XCD-contiguous order, TFLOP/s (a library
// product of the same sizes: 1340, 1070 and 1250):
//
//                                  32768 x 4096    4096 x 32768    4096 x 4096
//                                  x 4096          x 4096          x 32768
//   k of both operands contiguous  1380-1410
//   k of B outer (k of both)                       1340 (1250)
//   k of A outer                                                   1420
//   64-byte rows a slice, 4 slices 1240            1240 (both)     1330
//   the same without the phases    1080            920 (both)      960
//
// A z tile over 4096 entries keeps its CU busy for 168 000 cycles, of which the
// matrix cores work 131 000 (78%; dweight 68%, dhidden 70%), and under that load
// the clock stands at 1.8-1.9 GHz.  A loop of nothing but these instructions on
// random values reaches 2050 TFLOP/s at 2.0 GHz: most of the distance is matrix
// cores that wait, at a tile's ends and for the slices, the rest the clock.
template <int DT, bool AKO_, bool BKO_, int WM_ = 4>
struct RingProduct {
  static constexpr int MT = 256, NT = 256, NW = 8, WM = WM_, WN = NW / WM, MI = MT / WM / 16, NI = NT / WN / 16;
  static constexpr bool AKO = AKO_, BKO = BKO_;
  static constexpr int CHUNK = 16384, PLACES = 10;
  static constexpr int LDS_BYTES = CHUNK * PLACES;

  // Byte offset from the operand's slice of what lane `lane` loads in load j (0
  // ... 15) of chunk q (0, 1); *k: the first of its entries (k contiguous).
  template <bool KO>
  __device__ static __forceinline__ uint32_t load_offset(int q, int j, int lane, int32_t stride, int* k) {
    if constexpr (!KO) {
      const int r = j * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
      *k = c * 8;
      return ((uint32_t)(q * 128 + r) * (uint32_t)stride + c * 8) * 2;
    } else {
      const int kr = j * 2 + (lane >> 5), p = lane & 31;
      const int u = (p >> 1) ^ ((kr & 3) | (kr >> 1 & 4));
      *k = 0;
      return ((uint32_t)(q * 32 + kr) * (uint32_t)stride + u * 16 + (p & 1) * 8) * 2;
    }
  }

  // The fragment of rows r0 ... r0 + 15 (of the tile) and entries kk * 32 ... +
  // 31 of a slice whose first chunk of the operand lies at place `at`.
  template <bool KO>
  __device__ static __forceinline__ u32x4 fragment(lds_u16* chunk, int r0, int kk, int lane) {
    if constexpr (!KO) {
      const int r = (r0 & 127) + (lane & 15), c = kk * 4 + (lane >> 4);
      return *(__attribute__((address_space(3))) u32x4*)(chunk + r * 64 + (c ^ (r & 7)) * 8);
    } else {
      const int k = (lane >> 4) * 8 + ((lane & 15) >> 2);
      const int u = (r0 / 16) ^ ((k & 3) | (k >> 1 & 4));
      lds_u16* p = chunk + k * 256 + u * 16 + (lane & 3) * 4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * 256));
      const u32x2 l = __builtin_bit_cast(u32x2, lo), h = __builtin_bit_cast(u32x2, hi);
      return u32x4{l[0], l[1], h[0], h[1]};
    }
  }

  // one operand's way through its slices
  template <bool KO>
  struct Stream {
    const char* base;
    int64_t bytes, step;
    int32_t left;  // entries of k from the next slice on
    uint32_t off[4];
    int k[4];
    __device__ __forceinline__ Stream(const Operand& o, int32_t depth, int wave, int lane)
        : base((const char*)o.base), bytes(o.bytes), step(KO ? (int64_t)o.stride * 128 : 128), left(depth) {
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = load_offset<KO>(i >> 1, (i & 1) * 8 + wave, lane, o.stride, &k[i]);
    }
    // the next slice's two chunks to places p and p + 1; past the last slice nothing is in range
    __device__ __forceinline__ void load(lds_u16* lds, int p, int wave) {
      const int64_t n = left <= 0 || bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes;
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base, (uint32_t)n);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(lds + (p + (i >> 1)) * (CHUNK / 2) + ((i & 1) * 8 + wave) * 512),
            16, !KO && k[i] >= left ? kOOB : off[i], 0, 0, 0);
      base += step;
      bytes -= step;
      left -= 64;
    }
  };

  // acc <- A . B^T over k in [0, depth).
  __device__ static __forceinline__ void run(const Operand& a, const Operand& b, int32_t depth, uint16_t* lds_generic,
                                             f32x4 (&acc)[MI][NI]) {
    lds_u16* lds = (lds_u16*)lds_generic;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const bool late = wave >= NW / 2;
    Stream<AKO> sa(a, depth, wave, lane);
    Stream<BKO> sb(b, depth, wave, lane);
    const int32_t slices = (depth + 63) / 64;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    sa.load(lds, 0, wave);
    sb.load(lds, 2, wave);
    sa.load(lds, 4, wave);
    __builtin_amdgcn_s_waitcnt(wait_code(4));
    phase_end();
    if (late) phase_end();
    int p = 0;  // place of the slice's first chunk: always even, and its 4 chunks wrap in pairs
    for (int32_t t = 0; t < slices; ++t) {
      const int pb = p + 2 >= PLACES ? p + 2 - PLACES : p + 2;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 fa[MI], fb[NI];
        lds_u16* ca = lds + (p + (AKO ? kk : wm * MI >> 3)) * (CHUNK / 2);
        lds_u16* cb = lds + (pb + (BKO ? kk : wn * NI >> 3)) * (CHUNK / 2);
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[i] = fragment<AKO>(ca, (wm * MI + i) * 16, kk, lane);
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[j] = fragment<BKO>(cb, (wn * NI + j) * 16, kk, lane);
        __builtin_amdgcn_sched_barrier(0);
        if (kk == 0) {
          sb.load(lds, p + 6 >= PLACES ? p + 6 - PLACES : p + 6, wave);
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the fragments are here
        } else {
          sa.load(lds, p + 8 >= PLACES ? p + 8 - PLACES : p + 8, wave);
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(wait_code(4));  // ... and all of slice t + 1
        }
        phase_end();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = mfma16<DT>(fa[i], fb[j], acc[i][j]);
        __builtin_amdgcn_s_setprio(0);
        phase_end();
      }
      p = p + 4 >= PLACES ? p + 4 - PLACES : p + 4;
    }
    if (!late) phase_end();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_code(0));  // LDS is free again behind the next barrier
  }
};

// ---- a tile's way out ----------------------------------------------------------------
// A tile of 16-bit values on its way out: the fragments hold 4 neighbours of a
// row (of the output: a column of the product) a lane, which would store 32
// bytes of 16 rows at a time; through LDS whole rows of the tile go out, 16
// bytes a lane (dweight of one row, 131072 x 4096: 197 us, 311 with the
// fragments' own stores).  `from(mi, ni)` gives a fragment's 4 values as 8 bytes; `to(row)`
// is where a row of the tile begins, null if it does not exist, and `left` the
// elements from there on that do.
template <class P>
constexpr int kTileOutBytes = P::NT * (P::MT + 8) * 2;

template <class P, class From, class To>
__device__ __forceinline__ void tile_out(uint16_t* lds, int left, From&& from, To&& to) {
  constexpr int PITCH = P::MT + 8;  // 16 bytes off the banks' period
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / P::WN, wn = wave % P::WN;
  __syncthreads();  // the tile loop's LDS reads are over
#pragma unroll
  for (int ni = 0; ni < P::NI; ++ni)
#pragma unroll
    for (int mi = 0; mi < P::MI; ++mi)
      *(u32x2*)(lds + ((wn * P::NI + ni) * 16 + (lane & 15)) * PITCH + (wm * P::MI + mi) * 16 + (lane >> 4) * 4) =
          from(mi, ni);
  __syncthreads();
  constexpr int LPR = P::MT / 8;  // lanes of a row
  const int m = threadIdx.x % LPR * 8;
#pragma unroll 4
  for (int row = threadIdx.x / LPR; row < P::NT; row += P::NW * 64 / LPR) {
    uint16_t* p = to(row);
    if (!p || m >= left) continue;
    const u32x4 v = *(const u32x4*)(lds + row * PITCH + m);
    if (left - m >= 8) {
      *(u32x4_out*)(p + m) = v;
    } else {
      for (int j = 0; j < left - m; ++j) p[m + j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
    }
  }
}

// ---- tiles of a launch ------------------------------------------------------------------
// Tile (m, n) of workgroup b, false past the last one.  The hardware hands
// consecutive workgroups to the 8 XCDs in turn, so XCD k takes one contiguous
// run of tiles; in a run, `group` column tiles times some row tiles make the
// block of tiles that an XCD's 32 CUs work on at a time, which share their
// operands' slices in that XCD's L2.
__device__ __forceinline__ bool tile_of(int b, int mt, int nt, int group, int* m, int* n) {
  const int total = mt * nt, per = (total + 7) / 8;
  const int t = (b & 7) * per + (b >> 3);
  if ((b >> 3) >= per || t >= total) return false;
  const int g = t / (group * mt), r = t % (group * mt);
  const int w = nt - g * group < group ? nt - g * group : group;
  *m = r / w;
  *n = g * group + r % w;
  return true;
}

}  // namespace hprms
