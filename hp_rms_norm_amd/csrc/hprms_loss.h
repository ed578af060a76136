// hprms_loss.h - softmax cross entropy of rows under a vocabulary projection,
// without keeping the logits, and its gradient: device code.
//
// z = hidden . weight^T [rows, vocab];  lse = log(sum_v exp(z));
// loss = lse - z[target];  p = exp(z - lse);  dz = (p - [v == target]) * dloss;
// dhidden = dz . weight;  dweight = dz^T . hidden.
//
// Four matrix products on the matrix cores, each a tile loop whose epilogue
// does the rest:
//
//   forward   z tiles; each leaves per row its maximum and sum of exponentials
//             (and the target's logit); a second kernel joins the tiles.
//   gradient  for one piece of the vocabulary at a time: the z tiles again,
//             turned into dz, rounded to the tensors' 16-bit type and kept for
//             this piece only; then the piece's rows of dweight and its share of
//             dhidden, summed over the pieces in binary32.
//
// Rows whose target is ignore_index carry no loss: the others are listed first
// (`index`), the products run over the listed rows alone, and an ignored row's
// hidden values are never read.
//
// dz is rounded to 16 bits because the matrix cores take 16-bit operands: a
// relative error of half a step per entry, as the outputs' own rounding has.
// dloss is scaled first so that its largest magnitude is 2^14, and the products
// are scaled back in binary32: under one dloss for all rows, as a mean of losses
// has it, an entry's error then comes from p - 1 or p alone.  (Scaled by a power
// of two instead, that dloss's own rounding, up to half a step, was common to
// all entries of the targets: 0.0031 against 0.0023 relative error of the
// gradients at 500 rows.)  float16 holds dz down to probabilities of 2^-28; from
// there on it is subnormal, off by up to 2^-39 of the largest |dloss|, and a row
// whose dloss is 2^-k of the largest gets there at probabilities of 2^(k - 28).
// A scale for each row would serve such rows' dhidden, but dweight's sum over
// the rows would then need its inverse in hidden, the other float16 operand,
// which it would take below float16's normal numbers sooner.
//
// Fragments of v_mfma_f32_16x16x32: lane l holds A[l % 16][8 (l / 16) + j] and
// B[8 (l / 16) + j][l % 16], j = 0 ... 7, and of the product the four rows
// 4 (l / 16) + i of column l % 16.  The operand whose index should be
// contiguous in what the epilogue writes or reduces is A: the vocabulary for z,
// the hidden index for both gradients.  The tile loop: hprms_product.h.
#pragma once

#include "hprms_loss_rows.h"
#include "hprms_product.h"

namespace hprms {

// 8 bytes at any 2-byte boundary
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(2)));

// ---- epilogues ------------------------------------------------------------------------
// Each sees a wave's tile of MI x NI fragments whose first row and column are
// m and n (this lane's: + 16 mi + 4 (lane / 16) + i and + 16 ni + lane % 16).

__device__ __forceinline__ float xor16(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));
}
__device__ __forceinline__ float xor32(float v) { return __shfl_xor(v, 32); }

// exp(x) as 2^(x log2 e); the argument is at most 0 in every use but for NaN
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// The targets of this lane's columns, in the piece, or -1 (loaded before the
// tile loop: two dependent loads that would stand at its end).
template <int NI>
__device__ __forceinline__ void load_targets(const LossArgs& a, int n0, int wn, int count, int (&t)[NI]) {
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int n = n0 + (wn * NI + ni) * 16 + (threadIdx.x & 15);
    const int64_t in = n < count ? a.target[a.index[n]] - a.piece_from : -1;
    t[ni] = in >= 0 && in < a.piece ? (int)in : -1;
  }
}

// Per column (list position) of the workgroup's tile: the maximum over its
// vocabulary rows and the sum of exponentials relative to it.  A wave's 4 lanes
// of a column join by swizzles, the WM waves stacked over the column through
// LDS.  NaN logits leave the maximum and make the sum NaN.
// `t` is load_targets's.
template <int MI, int NI, int WM, int WN>
__device__ __forceinline__ void forward_epilogue(const LossArgs& a, const f32x4 (&acc)[MI][NI], const int (&t)[NI],
                                                 int m0, int n0, int wm, int wn, int count, int tile, float2* lds) {
  const int lane = threadIdx.x & 63;
  __syncthreads();  // the tile loop's LDS reads are over
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int col = wn * NI * 16 + ni * 16 + (lane & 15);
    const int n = n0 + col;
    float top = -__builtin_inff();
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = m0 + (wm * MI + mi) * 16 + (lane >> 4) * 4 + i;  // in the piece
        if (v < a.piece) top = fmaxf(top, acc[mi][ni][i]);
        if (v == t[ni]) a.target_logit[n] = acc[mi][ni][i];
      }
    top = fmaxf(top, xor16(top));
    top = fmaxf(top, xor32(top));
    const float at = top == -__builtin_inff() ? 0.0f : top;  // nothing but -inf here: every exponential is 0
    float sum = 0.0f;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = m0 + (wm * MI + mi) * 16 + (lane >> 4) * 4 + i;
        if (v < a.piece) sum += exp_neg(acc[mi][ni][i] - at);
      }
    sum += xor16(sum);
    sum += xor32(sum);
    if ((lane >> 4) == 0) lds[wm * (WN * NI * 16) + col] = float2{top, sum};
  }
  __syncthreads();
  for (int col = threadIdx.x; col < WN * NI * 16; col += WM * WN * 64) {
    if (n0 + col >= count) continue;
    float2 s = lds[col];
#pragma unroll
    for (int w = 1; w < WM; ++w) {
      const float2 o = lds[w * (WN * NI * 16) + col];
      const float top = fmaxf(s.x, o.x);
      const float at = top == -__builtin_inff() ? 0.0f : top;
      s = float2{top, s.y * exp_neg(s.x - at) + o.y * exp_neg(o.x - at)};
    }
    a.partial[(int64_t)tile * a.rows_at + (n0 + col - a.row_from)] = s;
  }
}

// The piece's dz of the tile, 0 where there is no row or no vocabulary entry.
// A target outside [0, vocab) gives NaN.
template <class P>
struct DzColumns {  // of this lane's columns; loaded before the tile loop, as in the forward kernel
  float lse[P::NI], g[P::NI];
  int t[P::NI];  // the target in the piece, or -1
  __device__ __forceinline__ void load(const LossArgs& a, int n0, int wn, int count) {
    const float scale = a.meta->scale;
#pragma unroll
    for (int ni = 0; ni < P::NI; ++ni) {
      const int n = n0 + (wn * P::NI + ni) * 16 + (threadIdx.x & 15);
      lse[ni] = g[ni] = 0.0f;
      t[ni] = -1;
      if (n < count) {
        const int row = a.index[n];
        const int64_t target = a.target[row];
        lse[ni] = a.lse[row];
        g[ni] = target >= 0 && target < a.vocab ? a.dloss[row] * scale : __builtin_nanf("");
        const int64_t in = target - a.piece_from;
        t[ni] = in >= 0 && in < a.piece ? (int)in : -1;
      }
    }
  }
};

template <class P, int DT>
__device__ __forceinline__ void dz_epilogue(const LossArgs& a, const f32x4 (&acc)[P::MI][P::NI], const DzColumns<P>& c,
                                            int m0, int n0, int count) {
  using F = Fmt<DT>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / P::WN, wn = wave % P::WN;
  // (through tile_out measured 3% slower here: 827 us against 802 for 4096 x 32768 x 4096)
#pragma unroll
  for (int ni = 0; ni < P::NI; ++ni) {
    const int n = n0 + (wn * P::NI + ni) * 16 + (lane & 15);
    uint16_t* to = a.dz + (int64_t)n * a.dz_stride;
#pragma unroll
    for (int mi = 0; mi < P::MI; ++mi) {
      const int m = m0 + (wm * P::MI + mi) * 16 + (lane >> 4) * 4;
      float d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = exp_neg(acc[mi][ni][i] - c.lse[ni]);
        d[i] = n < count && m + i < a.piece ? (m + i == c.t[ni] ? p - 1.0f : p) * c.g[ni] : 0.0f;
      }
      *(u32x2*)(to + m) = u32x2{F::pack(d[0], d[1]), F::pack(d[2], d[3])};
    }
  }
}

template <int DT>
__device__ __forceinline__ void store_four(uint16_t* p, const float* d, int n) {
  using F = Fmt<DT>;
  if (n >= 4) {
    *(u32x2_u*)p = u32x2_u{F::pack(d[0], d[1]), F::pack(d[2], d[3])};
  } else {
    for (int i = 0; i < n; ++i) p[i] = F::pack1(d[i]);
  }
}

// Rows of dweight: A is the hidden index, the column the vocabulary entry.
template <class P, int DT>
__device__ __forceinline__ void dweight_epilogue(const LossArgs& a, f32x4 (&acc)[P::MI][P::NI], int m0, int n0,
                                                 uint16_t* lds) {
  using F = Fmt<DT>;
  const float unscale = a.meta->unscale;
  tile_out<P>(
      lds, a.width - m0,
      [&](int mi, int ni) {
        const f32x4 d = acc[mi][ni] * unscale;
        return u32x2{F::pack(d[0], d[1]), F::pack(d[2], d[3])};
      },
      [&](int row) {
        return n0 + row < a.piece ? a.dweight + ((int64_t)a.piece_from + n0 + row) * a.dweight_stride + m0 : nullptr;
      });
}

// A piece's share of dhidden, or all of it: A is the hidden index, the column
// the list position.  With more than one share (pieces, or splits of a piece's
// vocabulary over workgroups) each goes to binary32 sums, which
// loss_dhidden_kernel adds up; a share's first piece sets its sum.
template <int DT, int MI, int NI>
__device__ __forceinline__ void dhidden_epilogue(const LossArgs& a, const f32x4 (&acc)[MI][NI], int m0, int n0, int wm,
                                                 int wn, int count, int split) {
  const int lane = threadIdx.x & 63;
  const float unscale = a.meta->unscale;
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int n = n0 + (wn * NI + ni) * 16 + (lane & 15);
    if (n >= count) continue;
    const int64_t row = a.sum ? 0 : a.index[n];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const int m = m0 + (wm * MI + mi) * 16 + (lane >> 4) * 4;
      if (a.sum) {
        if (m >= a.packed_width) continue;
        f32x4* s = (f32x4*)(a.sum + ((int64_t)split * count + n) * a.packed_width + m);
        *s = a.first_piece ? acc[mi][ni] : acc[mi][ni] + *s;
      } else if (m < a.width) {
        float d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = acc[mi][ni][i] * unscale;
        store_four<DT>(a.dhidden + row * a.dhidden_stride + m, d, a.width - m);
      }
    }
  }
}

}  // namespace hprms
