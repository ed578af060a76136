// hprms_norm_add_grad.hip - the gradient of the edge between two blocks
// (hprms_norm_add.hip): n = x * i(x) * post_weight, h = a * s + g * n, y = h *
// i(h) * weight, with i(v) = 1 / sqrt(mean(v^2) + eps).
//
// With d the gradient of y, e (optional) that of h by its other uses, h as the
// forward call stored it, r = i(h), q = i(x):
//
//   dh       = r * (d * weight) - h * (r^3 * mean(d * weight * h)) + e
//   ds       = a * dh
//   dweight  = sum over rows of d * h * r
//   dgate    = dh * n, summed over the rows that share the gate
//   dn       = g * dh
//   dpost    = sum over rows of dn * x * q
//   dx       = q * (dn * post_weight) - x * (q^3 * mean(dn * post_weight * x))
//
// (without post_weight dx = dn).  A row is read once, d, e, x, h and a gate of
// its own, and held in registers over two joins of its sums: three first (h^2,
// d * weight * h, x^2), then one that needs dh.  dx and ds are written: 6 rows of
// traffic a row, which HBM bounds.  A workgroup walks rows with a fixed step and
// keeps its lanes' columns of dweight, dpost and the gate's gradient in binary32
// registers; a second kernel adds the workgroups' rows of sums in a fixed order
// (no atomics: a call's bits do not change from run to run).
//
// A gate that rows share cuts the rows into units: all rows of a gate, or, where
// there are fewer gates than workgroups, an equal part of them.  A workgroup
// takes whole units and lets go of the gate's sums at each one's end, as a row
// of sums for the second kernel, or as the gradient itself where the unit is all
// of the gate's rows.  Units that are no multiple of the workgroups leave some of
// those idle: about 16 500 rows of 4096 take 147 us with 1 gate, 163 with 200, 164
// with 256, 205 with 129 and 241 with 257 (and, for a reason not looked for, 201
// with 64 and 235 with 128).
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_rows.h"

namespace hprms {
namespace {

struct NormAddGradArgs {
  const uint16_t* dout;
  const uint16_t* dresidual;  // null: none
  const uint16_t* input;
  const uint16_t* residual;     // as the forward call stored it
  const uint16_t* weight;
  const uint16_t* post_weight;  // null: none
  const uint16_t* gate;         // null: none
  uint16_t* dinput;
  uint16_t* dresidual_in;
  uint16_t* dgate;
  float* weight_sums;  // [gridDim.x, hidden]
  float* post_sums;    // [gridDim.x, hidden]
  float* gate_sums;    // [units, hidden] if parts > 1
  int64_t rows, gates, rows_per_gate, units;
  int32_t parts;      // units of a gate
  int64_t dout_stride, dresidual_stride, input_stride, residual_stride, gate_stride, dinput_stride,
      dresidual_in_stride, dgate_stride;
  int32_t hidden;
  float eps, residual_scale;
};

enum GateKind { kNoGate, kSharedGate, kElementGate };

// A lane's sums of its columns, N times 8: in registers, or (LDS) in its own slots
// of LDS.
template <bool LDS, int N, int BLOCK>
struct ColumnSums {
  float v[N][8];
  __device__ __forceinline__ void clear(int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
  }
  __device__ __forceinline__ void add(int i, const float (&t)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] += t[j];
  }
  __device__ __forceinline__ void get(int i, float (&t)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = v[i][j];
  }
};
template <int N, int BLOCK>
struct ColumnSums<true, N, BLOCK> {
  f32x4* at;
  __device__ __forceinline__ ColumnSums() {
    __shared__ f32x4 slots[2 * N * BLOCK];
    at = slots + threadIdx.x;
  }
  __device__ __forceinline__ void clear(int i) { at[2 * i * BLOCK] = at[(2 * i + 1) * BLOCK] = f32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void add(int i, const float (&t)[8]) {
    at[2 * i * BLOCK] += f32x4{t[0], t[1], t[2], t[3]};
    at[(2 * i + 1) * BLOCK] += f32x4{t[4], t[5], t[6], t[7]};
  }
  __device__ __forceinline__ void get(int i, float (&t)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = at[(2 * i + j / 4) * BLOCK][j % 4];
  }
};

// LPR lanes a row, VPL vectors of 8 elements a lane (slots as in hprms_rows.h).
// Per element and row, with m the product of what scales it behind dh (gate *
// post_weight, or the one there is):
//
//   first pass   squares of h and x, weight * (d * h)
//   second       dh; v = dh * x; z += q * v; sum of m * v; dweight += r * (d * h)
//   third        dx = q * (m * dh) - x * c
//
// z alone gives both columns' sums of a shared gate: its gradient is post_weight *
// z, and gate * z is its unit's share of dpost.  HOLD keeps weight and m as
// binary32 in registers (8 instructions an element fewer than unpacking them for
// each row), or weight and post_weight as they are (PACKED); LACC keeps the columns'
// sums in LDS.
template <int DT, int LPR, int VPL, int BLOCK, bool POST, int GATE, bool AHEAD, bool HOLD, bool LACC, bool NT>
__global__ __launch_bounds__(BLOCK) void norm_add_grad_kernel(NormAddGradArgs a) {
  constexpr int RPB = BLOCK / LPR;
  constexpr bool SHARED = GATE == kSharedGate, ELEMENT = GATE == kElementGate;
  constexpr bool SCALED = POST || SHARED;  // m is more than 1 (or a row's own gate)
  constexpr bool Z = POST || SHARED;
  // a row's own gate beside post_weight leaves no registers for both as binary32 (1021
  // x 5003: 36.1 us so, 32.3 with the two packed)
  constexpr bool PACKED = HOLD && ELEMENT && POST, FLOATS = HOLD && !PACKED;
  __shared__ float sums[2][BLOCK / 64 * 3];
  __shared__ float sums2[2][BLOCK / 64];
  __shared__ float cols[RPB > 1 ? RPB * LPR * 8 : 1];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  const int nvec = a.hidden >> 3, tail = a.hidden & 7;
  const int dup = tail ? 8 - tail : 0;  // the tail vector's elements that a whole vector holds
  int off[VPL], skip[VPL];
  bool on[VPL];
  u32x4 own[VPL];
  ColumnSums<LACC, (Z ? 2 : 1) * VPL, BLOCK> acc;  // dweight's, then z
  float* post_sums = a.post_sums + (int64_t)blockIdx.x * a.hidden;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int v = k * LPR + lane;
    on[k] = v < nvec + (tail ? 1 : 0);
    off[k] = v < nvec ? v * 8 : a.hidden - 8;
    skip[k] = v < nvec ? 0 : dup;
    own[k] = k >= VPL / 2 ? without_first(skip[k]) : without_first(0);
    acc.clear(k);
    if constexpr (Z) acc.clear(VPL + k);
  }
  // a column's sums over the row groups of the workgroup, in row group 0
  auto join = [&](float (&t)[8]) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) cols[(sub * LPR + lane) * 8 + j] = t[j];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int i = 1; i < RPB; ++i) t[j] += cols[(i * LPR + lane) * 8 + j];
      }
    }
  };
  auto put = [&](float* to, int k, const float (&t)[8]) {
    if (sub != 0 || !on[k]) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= skip[k]) to[off[k] + j] = t[j];
  };
  const u32x4 zeros = {0, 0, 0, 0};
  u32x4 nd[VPL], ne[VPL], nx[VPL], nh[VPL], ng[VPL];
  auto load = [&](int64_t row, bool in) {
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      nd[k] = ne[k] = nx[k] = nh[k] = ng[k] = zeros;
      if (in && on[k]) {
        nd[k] = load_row8_once<NT>(a.dout + row * a.dout_stride + off[k]);
        nh[k] = load_row8_once<NT>(a.residual + row * a.residual_stride + off[k]);
        nx[k] = load_row8_once<NT>(a.input + row * a.input_stride + off[k]);
        if (a.dresidual) ne[k] = load_row8_once<NT>(a.dresidual + row * a.dresidual_stride + off[k]);
        if constexpr (ELEMENT) ng[k] = load_row8(a.gate + row * a.gate_stride + off[k]);
      }
    }
  };
  const uint16_t* gate = a.gate;  // the unit's row of a shared one
  float wf[FLOATS ? VPL : 1][8], mf[FLOATS && SCALED ? VPL : 1][8];
  u32x4 wp[PACKED ? VPL : 1], pp[PACKED ? VPL : 1];
  auto vector = [&](const uint16_t* from, int k) {
    u32x4 v = on[k] ? load_row8(from + off[k]) : zeros;
    if (tail && k >= VPL / 2) v &= own[k];
    return v;
  };
  auto scales = [&](int k, float (&m)[8]) {
    const u32x4 p = PACKED ? pp[PACKED ? k : 0] : POST ? vector(a.post_weight, k) : zeros;
    const u32x4 g = SHARED ? vector(gate, k) : zeros;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      m[j] = POST && SHARED ? element<DT>(p, j) * element<DT>(g, j) : POST ? element<DT>(p, j) : element<DT>(g, j);
  };
  auto weights = [&](int k, float (&w)[8]) {
    const u32x4 v = PACKED ? wp[PACKED ? k : 0] : vector(a.weight, k);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = element<DT>(v, j);
  };
  if constexpr (HOLD) {
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      if constexpr (PACKED)
        wp[k] = vector(a.weight, k);
      else
        weights(k, wf[k]);
    }
  }
  int phase = 0;
  for (int64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
    // unit u is part u / gates of gate u % gates; a unit's rows are whole
    // workgroup steps, `parts` steps apart
    const int64_t at = SHARED ? unit % a.gates : 0;
    const int64_t part = SHARED ? unit / a.gates : unit;
    const int64_t end = SHARED ? (at + 1) * a.rows_per_gate : a.rows;
    const int64_t step = (int64_t)a.parts * RPB;
    const int64_t first = (SHARED ? at * a.rows_per_gate : 0) + part * RPB;
    if (first < end) load(first + sub, first + sub < end);
    if constexpr (SHARED) gate = a.gate + at * a.gate_stride;
    if constexpr (HOLD && SCALED) {
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        if constexpr (PACKED)
          pp[k] = vector(a.post_weight, k);  // (before the units: 8192 x 4096 112 us, 97 here)
        else
          scales(k, mf[k]);
      }
    }
    for (int64_t row0 = first; row0 < end; row0 += step) {
      const int64_t row = row0 + sub;
      const bool live = RPB == 1 || row < end;
      u32x4 d[VPL], e[VPL], x[VPL], h[VPL], g[VPL];
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        d[k] = nd[k];
        e[k] = ne[k];
        x[k] = nx[k];
        h[k] = nh[k];
        g[k] = ng[k];
        if (tail && k >= VPL / 2) {
          d[k] &= own[k];
          e[k] &= own[k];
          x[k] &= own[k];
          h[k] &= own[k];
          g[k] &= own[k];
        }
      }
      if constexpr (AHEAD) load(row + step, row + step < end);
      float s[POST ? 3 : 2] = {};
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        float w[8];
        if constexpr (!FLOATS) weights(k, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float hf = element<DT>(h[k], j);
          s[0] += hf * hf;
          s[1] += (element<DT>(d[k], j) * hf) * (FLOATS ? wf[FLOATS ? k : 0][j] : w[j]);
          if constexpr (POST) s[2] += element<DT>(x[k], j) * element<DT>(x[k], j);
        }
        packed_again(d[k]);
        packed_again(x[k]);
        packed_again(h[k]);
      }
      sum_rows<POST ? 3 : 2, LPR, BLOCK>(s, sums[phase]);
      const float n = (float)a.hidden;
      // (a row group without a row holds zeros, and adds zeros to the columns' sums)
      const float r = live ? 1.0f / sqrtf(s[0] / n + a.eps) : 0.0f;
      const float rc = r * r * (r * (s[1] / n));
      const float q = !POST ? 1.0f : live ? 1.0f / sqrtf(s[POST ? 2 : 0] / n + a.eps) : 0.0f;
      float mv[1] = {0.0f};
      float u[POST ? VPL : 1][8];
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        float w[8], m[8], o[8], dx[8], dg[8], tw[8], tz[8];
        if constexpr (PACKED) {
          packed_again(wp[k]);
          packed_again(pp[k]);
        }
        if constexpr (!FLOATS) weights(k, w);
        if constexpr (!FLOATS && SCALED) scales(k, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float hf = element<DT>(h[k], j), df = element<DT>(d[k], j), xf = element<DT>(x[k], j);
          const float wj = FLOATS ? wf[FLOATS ? k : 0][j] : w[j];
          float dh = r * (df * wj) - hf * rc + element<DT>(e[k], j);
          o[j] = dh * a.residual_scale;
          tw[j] = (df * hf) * r;
          float v = dh * xf;  // q times this: what the first norm passes on, without its weight
          if constexpr (SCALED) {
            const float mj = FLOATS ? mf[FLOATS && SCALED ? k : 0][j] : m[j];
            if constexpr (ELEMENT) {
              // gate * post_weight first, as a shared gate has it (in binary32 exact): a
              // row's bits are the same whichever kind its gate is
              const float gf = element<DT>(g[k], j), mg = mj * gf;
              dg[j] = (v * q) * mj;
              tz[j] = (v * gf) * q;
              mv[0] += v * mg;
              dh *= mg;
            } else {
              tz[j] = v * q;
              mv[0] += v * mj;
              dh *= mj;
            }
          } else if constexpr (ELEMENT) {
            dg[j] = v;
            dh *= element<DT>(g[k], j);
          }
          if constexpr (POST)
            u[k][j] = dh;
          else
            dx[j] = dh;
        }
        acc.add(k, tw);
        if constexpr (Z) acc.add(VPL + k, tz);
        if (live && on[k]) {
          store_row8(a.dresidual_in + row * a.dresidual_in_stride + off[k], pack8<DT>(o), skip[k]);
          if constexpr (ELEMENT) store_row8(a.dgate + row * a.dgate_stride + off[k], pack8<DT>(dg), skip[k]);
          if constexpr (!POST) store_row8(a.dinput + row * a.dinput_stride + off[k], pack8<DT>(dx), skip[k]);
        }
        packed_again(x[k]);
      }
      if constexpr (POST) {
        sum_rows<1, LPR, BLOCK>(mv, sums2[phase]);
        const float c = q * q * (q * (mv[0] / n));
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
          float dx[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) dx[j] = q * u[k][j] - element<DT>(x[k], j) * c;
          if (live && on[k])
            store_row8(a.dinput + row * a.dinput_stride + off[k], pack8<DT>(dx), skip[k]);
        }
      }
      phase ^= 1;
      if constexpr (!AHEAD) load(row + step, row + step < end);
    }
    if constexpr (SHARED) {
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        float t[8];
        acc.get(VPL + k, t);
        acc.clear(VPL + k);
        const u32x4 p = POST && on[k] ? load_row8(a.post_weight + off[k]) : zeros;
        if constexpr (POST) {
          const u32x4 g = on[k] ? load_row8(gate + off[k]) : zeros;
          float share[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            share[j] = t[j] * element<DT>(g, j);
            t[j] *= element<DT>(p, j);
          }
          join(share);
          // the workgroup's row of sums of dpost grows by each of its units
          if (unit >= gridDim.x && sub == 0 && on[k]) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j >= skip[k]) share[j] += post_sums[off[k] + j];
          }
          put(post_sums, k, share);
        }
        join(t);
        if (a.parts > 1)
          put(a.gate_sums + unit * a.hidden, k, t);
        else if (sub == 0 && on[k])
          store_row8(a.dgate + at * a.dgate_stride + off[k], pack8<DT>(t), skip[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    float t[8];
    acc.get(k, t);
    join(t);
    put(a.weight_sums + (int64_t)blockIdx.x * a.hidden, k, t);
    if constexpr (POST && !SHARED) {
      acc.get(VPL + k, t);
      join(t);
      put(post_sums, k, t);
    }
  }
}

// ---- any width: passes over the rows ---------------------------------------------------
// Rows of fewer than 8 or more than 16384 elements.  First what a row's elements
// share, {r, r^3 mean(d weight h), q, q^3 mean(dn post x)}; then the columns' sums,
// before the rows are written, which may lie on those that are read.
struct AnyRow {
  const uint16_t *d, *e, *x, *h, *g;
  __device__ __forceinline__ AnyRow(const NormAddGradArgs& a, int64_t row)
      : d(a.dout + row * a.dout_stride), e(a.dresidual ? a.dresidual + row * a.dresidual_stride : nullptr),
        x(a.input + row * a.input_stride), h(a.residual + row * a.residual_stride),
        g(a.gate ? a.gate + row / a.rows_per_gate * a.gate_stride : nullptr) {}
  template <class F>
  __device__ __forceinline__ float dh(const NormAddGradArgs& a, int64_t i, f32x4 f) const {
    const float v = f[0] * (F::one(d[i]) * F::one(a.weight[i])) - F::one(h[i]) * f[1];
    return e ? v + F::one(e[i]) : v;
  }
};

template <int DT>
__global__ __launch_bounds__(256) void norm_add_grad_factors_kernel(NormAddGradArgs a, f32x4* factors) {
  using F = Fmt<DT>;
  __shared__ float sums[12], sums2[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const AnyRow in(a, row);
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (int32_t i = threadIdx.x; i < a.hidden; i += 256) {
      const float h = F::one(in.h[i]), x = F::one(in.x[i]);
      s[0] += h * h;
      s[1] += F::one(in.d[i]) * F::one(a.weight[i]) * h;
      s[2] += x * x;
    }
    __syncthreads();
    sum_rows<3, 256, 256>(s, sums);
    const float n = (float)a.hidden, r = 1.0f / sqrtf(s[0] / n + a.eps);
    f32x4 f = {r, r * r * (r * (s[1] / n)), a.post_weight ? 1.0f / sqrtf(s[2] / n + a.eps) : 1.0f, 0.0f};
    if (a.post_weight) {
      float u[1] = {0.0f};
      for (int32_t i = threadIdx.x; i < a.hidden; i += 256) {
        float t = in.dh<F>(a, i, f);
        if (in.g) t *= F::one(in.g[i]);
        u[0] += t * F::one(a.post_weight[i]) * F::one(in.x[i]);
      }
      sum_rows<1, 256, 256>(u, sums2);
      f[3] = f[2] * f[2] * (f[2] * (u[0] / n));
    }
    if (threadIdx.x == 0) factors[row] = f;
  }
}

// Units as above, one a workgroup row (blockIdx.y): a column's sums over its rows.
template <int DT>
__global__ __launch_bounds__(256) void norm_add_grad_columns_kernel(NormAddGradArgs a, const f32x4* factors,
                                                                    bool shared) {
  using F = Fmt<DT>;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.hidden) return;
  float aw = 0.0f, ap = 0.0f;
  for (int64_t unit = blockIdx.y; unit < a.units; unit += gridDim.y) {
    const int64_t gate = shared ? unit % a.gates : 0, part = shared ? unit / a.gates : unit;
    const int64_t end = shared ? (gate + 1) * a.rows_per_gate : a.rows;
    float ag = 0.0f;
    for (int64_t row = (shared ? gate * a.rows_per_gate : 0) + part; row < end; row += a.parts) {
      const AnyRow in(a, row);
      const f32x4 f = factors[row];
      const float dh = in.dh<F>(a, i, f), nx = F::one(in.x[i]) * f[2];
      aw += F::one(in.d[i]) * (F::one(in.h[i]) * f[0]);
      ap += (in.g ? dh * F::one(in.g[i]) : dh) * nx;
      ag += dh * (a.post_weight ? nx * F::one(a.post_weight[i]) : nx);
    }
    if (shared && a.parts > 1)
      a.gate_sums[unit * a.hidden + i] = ag;
    else if (shared)
      a.dgate[gate * a.dgate_stride + i] = F::pack1(ag);
  }
  a.weight_sums[(int64_t)blockIdx.y * a.hidden + i] = aw;
  if (a.post_weight) a.post_sums[(int64_t)blockIdx.y * a.hidden + i] = ap;
}

template <int DT>
__global__ __launch_bounds__(256) void norm_add_grad_rows_kernel(NormAddGradArgs a, const f32x4* factors,
                                                                 bool element_gate) {
  using F = Fmt<DT>;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const AnyRow in(a, row);
    const f32x4 f = factors[row];
    for (int32_t i = threadIdx.x; i < a.hidden; i += 256) {
      const float dh = in.dh<F>(a, i, f), x = F::one(in.x[i]);
      float t = in.g ? dh * F::one(in.g[i]) : dh;
      float n = x;
      if (a.post_weight) {
        const float p = F::one(a.post_weight[i]);
        n = x * f[2] * p;
        t = f[2] * (t * p) - x * f[3];
      }
      a.dresidual_in[row * a.dresidual_in_stride + i] = F::pack1(dh * a.residual_scale);
      a.dinput[row * a.dinput_stride + i] = F::pack1(t);
      if (element_gate) a.dgate[row * a.dgate_stride + i] = F::pack1(dh * n);
    }
  }
}

// ---- the rows of sums ----------------------------------------------------------------------
// Output blockIdx.y: 0 dweight, 1 dpost, 2 ... the gates' (output row g: rows of
// sums g, g + gates, ...).  32 columns a workgroup, its 32 row lanes' sums added in
// order.
struct SumsOut {
  const float* sums;
  void* out;
  int32_t dtype;
};
struct JoinArgs {
  SumsOut weight, post, gate;
  int32_t rows, gate_parts, hidden;
  int64_t gates, gate_stride;
};

__global__ __launch_bounds__(1024) void norm_add_grad_join_kernel(JoinArgs a, int64_t from) {
  __shared__ float lds[32][33];
  const int64_t y = from + blockIdx.y;
  const SumsOut o = y == 0 ? a.weight : y == 1 ? a.post : a.gate;
  if (!o.out) return;
  const int64_t gate = y < 2 ? 0 : y - 2, step = y < 2 ? 1 : a.gates;
  const int32_t parts = y < 2 ? a.rows : a.gate_parts;
  const int c = threadIdx.x & 31, p = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float acc = 0.0f;
  if (col < a.hidden) {
    constexpr int U = 8;  // loads on their way at once
    for (int64_t i = p; i < parts; i += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = i + 32 * u < parts ? o.sums[(gate + (i + 32 * u) * step) * a.hidden + col] : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) acc += v[u];
    }
  }
  lds[p][c] = acc;
  __syncthreads();
  if (p != 0 || col >= a.hidden) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) acc += lds[i][c];
  const int64_t at = gate * (y < 2 ? 0 : a.gate_stride) + col;
  if (o.dtype == HPRMS_DTYPE_FP32)
    ((float*)o.out)[at] = acc;
  else
    ((uint16_t*)o.out)[at] =
        o.dtype == HPRMS_DTYPE_BF16 ? Fmt<HPRMS_DTYPE_BF16>::pack1(acc) : Fmt<HPRMS_DTYPE_FP16>::pack1(acc);
}

// ---- host ------------------------------------------------------------------------------
constexpr int64_t kMaxHidden = int64_t(1) << 24;
constexpr int64_t kVectorHidden = 16384;  // the register-resident kernels' widest rows

// Shapes by width.  Up to 8192 elements a workgroup of 8 waves a CU, 2 vectors a
// lane where the width has them, with the next rows' loads ahead and weights and
// sums in registers.  Times on bf16 rows with dresidual and one gate for all (none
// up to 512), both kernels, lanes x vectors x workgroup x workgroups per CU (33.5 M
// elements, 403 MB): 128 16 x 1 x 512 x 2 83.1 us, 16 x 1 x 256 x 4 87.7; 256 32 x
// 1 x 512 x 2 77.3, 64 x 1 96.3; 512 32 x 2 x 512 x 1 78.0, 64 x 1 82.2; 1024 64 x
// 2 x 512 x 1 77.0, x 256 x 2 78.6, 128 x 2 87.6; 2048 128 x 2 x 512 x 1 78.0, x
// 256 x 2 84.4, 256 x 2 90.0; 4096 256 x 2 x 512 x 1 81.6, 512 x 1 x 512 x 2 96.9,
// 512 x 1 x 1024 x 1 94.6; 8192 512 x 2 x 512 x 1 90.2, 1024 x 1 105.  Without the
// loads ahead 4096 takes 99.3, with weights unpacked for each row 108.  Past 8192
// the registers hold neither the sums (they lie in LDS) nor a second row: 16384
// 512 x 4 135.6 us, 1024 x 2 138.4, sums in registers 224 (120 to 180 spilled).
struct Shape {
  int lpr, vpl, block, per_cu;
};

Shape shape_of(int64_t hidden) {
  const int64_t slots = (hidden + 7) / 8;
  if (slots <= 16) return {16, 1, 512, 2};
  if (slots <= 32) return {32, 1, 512, 2};
  if (slots <= 64) return {32, 2, 512, 1};
  if (slots <= 128) return {64, 2, 512, 1};
  if (slots <= 256) return {128, 2, 512, 1};
  if (slots <= 512) return {256, 2, 512, 1};
  if (slots <= 1024) return {512, 2, 512, 1};
  return {512, 4, 512, 1};
}

bool is_general(int64_t hidden) { return hidden < 8 || hidden > kVectorHidden; }

struct Plan {
  int64_t grid, units, gates;
  int32_t parts;
  bool shared, element;
  int64_t post_sums, gate_sums, factors, total;  // byte offsets; weight_sums at 0
};

// gate_rows: 0 without a gate, else the gate's rows
Plan plan_of(int64_t rows, int64_t hidden, int64_t gate_rows, bool post) {
  Plan p = {};
  const bool general = is_general(hidden);
  const Shape s = general ? Shape{1, 1, 1, 0} : shape_of(hidden);
  const int64_t rpb = s.block / s.lpr;
  const int64_t most = general ? 64 : (int64_t)current_cus() * s.per_cu;
  // (the general path's columns kernel writes a shared gate's gradient before its rows kernel reads the
  // gate, on which dgate may lie where every row has its own: there one row is such a case too)
  p.element = gate_rows > 0 && gate_rows == rows && (rows > 1 || general);
  p.shared = gate_rows > 0 && !p.element;
  p.gates = p.shared ? gate_rows : 1;
  if (rows > 0) {
    const int64_t groups = (rows / p.gates + rpb - 1) / rpb;  // steps of a workgroup over a gate's rows
    p.parts = (int32_t)(p.gates >= most ? 1 : most / p.gates < groups ? most / p.gates : groups);
    p.units = p.gates * p.parts;
    p.grid = p.units < most ? p.units : most;
  }
  const int64_t row_bytes = (hidden * 4 + 15) & ~int64_t(15);
  int64_t at = p.grid * row_bytes;
  p.post_sums = at;
  if (post) at += p.grid * row_bytes;
  p.gate_sums = at;
  if (p.shared && p.parts > 1) at += p.units * row_bytes;
  p.factors = at;
  if (general) at += rows * 16;
  p.total = at;
  return p;
}

template <int DT, int LPR, int VPL, int BLOCK, bool AHEAD, bool HOLD, bool LACC, bool POST, bool NT>
void launch_gate(const NormAddGradArgs& a, const Plan& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.grid), block(BLOCK);
  if (p.element)
    norm_add_grad_kernel<DT, LPR, VPL, BLOCK, POST, kElementGate, AHEAD, HOLD, LACC, NT><<<grid, block, 0, stream>>>(a);
  else if (p.shared)
    norm_add_grad_kernel<DT, LPR, VPL, BLOCK, POST, kSharedGate, AHEAD, HOLD, LACC, NT><<<grid, block, 0, stream>>>(a);
  else
    norm_add_grad_kernel<DT, LPR, VPL, BLOCK, POST, kNoGate, AHEAD, HOLD, LACC, NT><<<grid, block, 0, stream>>>(a);
}

template <int DT, int LPR, int VPL, int BLOCK, bool AHEAD, bool HOLD, bool LACC>
void launch_rows(const NormAddGradArgs& a, const Plan& p, hipStream_t stream) {
  const bool nt = past_caches(a.rows, a.hidden,
                              {{a.dout, a.dout_stride},
                               {a.residual, a.residual_stride},
                               {a.input, a.input_stride},
                               {a.dresidual, a.dresidual ? a.dresidual_stride : 0}});
  if (a.post_weight && nt)
    launch_gate<DT, LPR, VPL, BLOCK, AHEAD, HOLD, LACC, true, true>(a, p, stream);
  else if (a.post_weight)
    launch_gate<DT, LPR, VPL, BLOCK, AHEAD, HOLD, LACC, true, false>(a, p, stream);
  else if (nt)
    launch_gate<DT, LPR, VPL, BLOCK, AHEAD, HOLD, LACC, false, true>(a, p, stream);
  else
    launch_gate<DT, LPR, VPL, BLOCK, AHEAD, HOLD, LACC, false, false>(a, p, stream);
}

template <int DT>
void launch_all(const NormAddGradArgs& a, const Plan& p, char* ws, hipStream_t stream) {
  if (is_general(a.hidden)) {
    f32x4* factors = (f32x4*)(ws + p.factors);
    const unsigned rows = (unsigned)(a.rows < 4096 ? a.rows : 4096);
    norm_add_grad_factors_kernel<DT><<<dim3(rows), dim3(256), 0, stream>>>(a, factors);
    norm_add_grad_columns_kernel<DT><<<dim3((unsigned)((a.hidden + 255) / 256), (unsigned)p.grid), dim3(256), 0,
                                       stream>>>(a, factors, p.shared);
    norm_add_grad_rows_kernel<DT><<<dim3(rows), dim3(256), 0, stream>>>(a, factors, p.element);
    return;
  }
  const Shape s = shape_of(a.hidden);
  switch (s.lpr * 8 + s.vpl) {
    case 16 * 8 + 1: launch_rows<DT, 16, 1, 512, true, true, false>(a, p, stream); break;
    case 32 * 8 + 1: launch_rows<DT, 32, 1, 512, true, true, false>(a, p, stream); break;
    case 32 * 8 + 2: launch_rows<DT, 32, 2, 512, true, true, false>(a, p, stream); break;
    case 64 * 8 + 2: launch_rows<DT, 64, 2, 512, true, true, false>(a, p, stream); break;
    case 128 * 8 + 2: launch_rows<DT, 128, 2, 512, true, true, false>(a, p, stream); break;
    case 256 * 8 + 2: launch_rows<DT, 256, 2, 512, true, true, false>(a, p, stream); break;
    case 512 * 8 + 2: launch_rows<DT, 512, 2, 512, true, true, false>(a, p, stream); break;
    default: launch_rows<DT, 512, 4, 512, false, false, true>(a, p, stream); break;
  }
}

int check_sizes(int64_t rows, int64_t hidden, int64_t gate_rows) {
  if (rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)rows);
  if (hidden < 1) return fail(HPRMS_E_INVALID, "hidden must be >= 1 (got %lld)", (long long)hidden);
  if (hidden > kMaxHidden)
    return fail(HPRMS_E_RANGE, "hidden %lld exceeds the supported maximum %lld", (long long)hidden,
                (long long)kMaxHidden);
  if (rows >= int64_t(1) << 31) return fail(HPRMS_E_RANGE, "rows %lld exceed 2^31 - 1", (long long)rows);
  if (gate_rows < 0 || gate_rows >= int64_t(1) << 31 || (gate_rows > 0 && rows % gate_rows != 0))
    return fail(HPRMS_E_INVALID, "gate_rows must divide rows (got %lld of %lld)", (long long)gate_rows,
                (long long)rows);
  return HPRMS_OK;
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_norm_add_rmsnorm_backward_workspace(int64_t rows, int64_t hidden, int64_t gate_rows) {
  const int rc = check_sizes(rows, hidden, gate_rows);
  return rc != HPRMS_OK ? rc : plan_of(rows, hidden, gate_rows, true).total;
}

int hprms_norm_add_rmsnorm_backward(void* dinput, void* dresidual_in, void* dpost_weight, void* dweight, void* dgate,
                                    const void* dout, const void* dresidual, const void* input, const void* residual,
                                    const void* post_weight, const void* weight, const void* gate, void* workspace,
                                    int64_t workspace_size, int64_t rows, int64_t hidden, int64_t gate_rows,
                                    int64_t dinput_row_stride, int64_t dresidual_in_row_stride,
                                    int64_t dgate_row_stride, int64_t dout_row_stride, int64_t dresidual_row_stride,
                                    int64_t input_row_stride, int64_t residual_row_stride, int64_t gate_row_stride,
                                    int dtype, int dpost_weight_dtype, int dweight_dtype, double residual_scale,
                                    double eps, hipStream_t stream) {
  if (dtype != HPRMS_DTYPE_BF16 && dtype != HPRMS_DTYPE_FP16)
    return fail(HPRMS_E_INVALID, "dtype must be HPRMS_DTYPE_BF16 or HPRMS_DTYPE_FP16 (got %d)", dtype);
  if ((dweight_dtype != dtype && dweight_dtype != HPRMS_DTYPE_FP32) ||
      (post_weight && dpost_weight_dtype != dtype && dpost_weight_dtype != HPRMS_DTYPE_FP32))
    return fail(HPRMS_E_INVALID, "dweight_dtype and dpost_weight_dtype must be dtype or HPRMS_DTYPE_FP32 (got %d, %d)",
                dweight_dtype, dpost_weight_dtype);
  if (!gate) gate_rows = 0;
  const int rc = check_sizes(rows, hidden, gate_rows);
  if (rc != HPRMS_OK) return rc;
  if (gate && gate_rows < 1 && rows > 0) return fail(HPRMS_E_INVALID, "a gate needs gate_rows >= 1");
  if (dinput_row_stride < hidden || dresidual_in_row_stride < hidden || dout_row_stride < hidden ||
      input_row_stride < hidden || residual_row_stride < hidden || (dresidual && dresidual_row_stride < hidden) ||
      (gate && (gate_row_stride < hidden || dgate_row_stride < hidden)))
    return fail(HPRMS_E_INVALID, "row strides must be >= hidden");
  if (!(eps >= 0.0)) return fail(HPRMS_E_INVALID, "eps must be >= 0");
  if (!(residual_scale - residual_scale == 0.0)) return fail(HPRMS_E_INVALID, "residual_scale must be finite");
  for (int64_t stride : {dinput_row_stride, dresidual_in_row_stride, dout_row_stride, input_row_stride,
                         residual_row_stride, dresidual ? dresidual_row_stride : hidden})
    if (!extent_ok(rows, stride, 2, hidden))
      return fail(HPRMS_E_RANGE, "%lld rows at these row strides span more than 2^56 bytes", (long long)rows);
  if (gate && (!extent_ok(gate_rows, gate_row_stride, 2, hidden) || !extent_ok(gate_rows, dgate_row_stride, 2, hidden)))
    return fail(HPRMS_E_RANGE, "the gate's rows at these strides span more than 2^56 bytes");
  if (!dweight || (post_weight && !dpost_weight) || (gate && !dgate) ||
      (rows > 0 && (!dinput || !dresidual_in || !dout || !input || !residual || !weight)))
    return fail(HPRMS_E_INVALID, "null tensor pointer");
  if ((((uintptr_t)dinput | (uintptr_t)dresidual_in | (uintptr_t)dgate | (uintptr_t)dout | (uintptr_t)dresidual |
        (uintptr_t)input | (uintptr_t)residual | (uintptr_t)post_weight | (uintptr_t)weight | (uintptr_t)gate |
        (uintptr_t)dweight | (uintptr_t)dpost_weight) & 1) != 0 ||
      (dweight_dtype == HPRMS_DTYPE_FP32 && ((uintptr_t)dweight & 3) != 0) ||
      (post_weight && dpost_weight_dtype == HPRMS_DTYPE_FP32 && ((uintptr_t)dpost_weight & 3) != 0))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  if (rows > 0 && dinput == dresidual_in)
    return fail(HPRMS_E_INVALID, "dinput and dresidual_in alias each other");
  // a row is read before it is written, by the workgroup that has it
  auto moves = [&](const void* out, int64_t out_stride, const void* in, int64_t in_stride) {
    return in && out == in && rows > 1 && out_stride != in_stride;
  };
  if (moves(dinput, dinput_row_stride, dout, dout_row_stride) ||
      moves(dinput, dinput_row_stride, dresidual, dresidual_row_stride) ||
      moves(dinput, dinput_row_stride, input, input_row_stride) ||
      moves(dinput, dinput_row_stride, residual, residual_row_stride) ||
      moves(dresidual_in, dresidual_in_row_stride, dout, dout_row_stride) ||
      moves(dresidual_in, dresidual_in_row_stride, dresidual, dresidual_row_stride) ||
      moves(dresidual_in, dresidual_in_row_stride, input, input_row_stride) ||
      moves(dresidual_in, dresidual_in_row_stride, residual, residual_row_stride) ||
      moves(dgate, dgate_row_stride, gate, gate_row_stride))
    return fail(HPRMS_E_INVALID, "an in-place alias needs equal row strides");
  if (rows > 0 && gate && dgate == gate && gate_rows != rows)
    return fail(HPRMS_E_INVALID, "dgate aliases a gate that rows share");
  const Plan p = plan_of(rows, hidden, gate_rows, post_weight != nullptr);
  if (p.total > 0 && (!workspace || workspace_size < p.total || ((uintptr_t)workspace & 15) != 0))
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 16-byte aligned (got %lld)", (long long)p.total,
                (long long)workspace_size);
  char* ws = (char*)workspace;
  NormAddGradArgs a = {};
  a.dout = (const uint16_t*)dout;
  a.dresidual = (const uint16_t*)dresidual;
  a.input = (const uint16_t*)input;
  a.residual = (const uint16_t*)residual;
  a.weight = (const uint16_t*)weight;
  a.post_weight = (const uint16_t*)post_weight;
  a.gate = (const uint16_t*)gate;
  a.dinput = (uint16_t*)dinput;
  a.dresidual_in = (uint16_t*)dresidual_in;
  a.dgate = (uint16_t*)dgate;
  a.weight_sums = (float*)ws;
  a.post_sums = (float*)(ws + p.post_sums);
  a.gate_sums = (float*)(ws + p.gate_sums);
  a.rows = rows;
  a.gates = p.gates;
  a.rows_per_gate = gate_rows > 0 && rows > 0 ? rows / gate_rows : 1;
  a.units = p.units;
  a.parts = p.parts;
  a.dout_stride = dout_row_stride;
  a.dresidual_stride = dresidual_row_stride;
  a.input_stride = input_row_stride;
  a.residual_stride = residual_row_stride;
  a.gate_stride = gate_row_stride;
  a.dinput_stride = dinput_row_stride;
  a.dresidual_in_stride = dresidual_in_row_stride;
  a.dgate_stride = dgate_row_stride;
  a.hidden = (int32_t)hidden;
  a.eps = (float)eps;
  a.residual_scale = (float)residual_scale;
  if (rows > 0) {
    if (dtype == HPRMS_DTYPE_BF16)
      launch_all<HPRMS_DTYPE_BF16>(a, p, ws, stream);
    else
      launch_all<HPRMS_DTYPE_FP16>(a, p, ws, stream);
  }
  // rows == 0: no rows of sums, and every sum is the empty one
  JoinArgs j = {};
  j.weight = {a.weight_sums, dweight, dweight_dtype};
  if (post_weight) j.post = {a.post_sums, dpost_weight, dpost_weight_dtype};
  j.rows = (int32_t)p.grid;
  j.hidden = a.hidden;
  j.gates = gate ? (rows > 0 ? p.gates : gate_rows) : 0;
  j.gate_stride = dgate_row_stride;
  const bool join_gates = gate && (rows == 0 || (p.shared && p.parts > 1));
  if (join_gates) {
    j.gate = {a.gate_sums, dgate, dtype};
    j.gate_parts = rows > 0 ? p.parts : 0;
  }
  const int64_t outputs = 2 + (join_gates ? j.gates : 0);
  for (int64_t from = 0; from < outputs; from += 32768)
    norm_add_grad_join_kernel<<<dim3((unsigned)((hidden + 31) / 32),
                                     (unsigned)(outputs - from < 32768 ? outputs - from : 32768)),
                                dim3(1024), 0, stream>>>(j, from);
  return check_launch("norm + gate + add + norm gradient kernel");
}

}  // extern "C"
