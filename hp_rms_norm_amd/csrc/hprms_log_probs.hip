// hprms_log_probs.hip - log probabilities of given tokens under rows of logits, with
// the entropy and the most likely alternatives, and the gradient.
//
//   m = max z;  S = sum e^(z - m);  lse = m + log S;  log_prob = z[token] - lse
//   entropy = log S + (sum e^(z - m) (m - z)) / S      (all terms >= 0)
//   top alternatives: the largest z, equal ones by the lower index, minus lse
//   dz = dlog_prob * ([v == token] - p) - dentropy * p * (log p + entropy)
//
// Forward, first kernel: a workgroup takes a part of a row, up to kPartBytes of it,
// into registers at once, 16 bytes a lane and step, and leaves the part's m, S and
// sum of e^(z - m) (z - m) and its `top` largest as sorted keys: its loads are all
// on their way before the first is used, and the logits are read once.  Second
// kernel: a wave joins a row's parts; a row of one part needs none.  The gradient
// is one pass over the logits, from the forward call's lse and entropy.
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_rows.h"

namespace hprms {
namespace {

typedef unsigned long long u64;

constexpr int kSteps = 16;                 // 16-byte loads of a lane, at most
constexpr int kStepBytes = 256 * 16;       // of a workgroup
constexpr int kPartBytes = kSteps * kStepBytes;  // 32768 16-bit or 16384 32-bit logits
constexpr int kMaxParts = 64;
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
// exponents of 2 below this give 0; bounds what 0 is multiplied with at -infinity
constexpr float kLowest = -200.0f;

template <int DT>
struct Logits {
  static constexpr int N = DT == HPRMS_DTYPE_FP32 ? 4 : 8;  // of a vector
  static constexpr int SIZE = DT == HPRMS_DTYPE_FP32 ? 4 : 2;
  static constexpr int LAST_BIT = DT == HPRMS_DTYPE_FP32 ? 0 : DT == HPRMS_DTYPE_BF16 ? 16 : 13;  // as binary32
  static constexpr uint32_t MINUS_INF =
      DT == HPRMS_DTYPE_FP32 ? 0xff800000u : DT == HPRMS_DTYPE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  __device__ static __forceinline__ float get(const u32x4& v, int j) {
    if constexpr (DT == HPRMS_DTYPE_FP32)
      return __uint_as_float(v[j]);
    else
      return element<DT>(v, j);
  }
  __device__ static __forceinline__ float one(const char* p) {
    if constexpr (DT == HPRMS_DTYPE_FP32)
      return *(const float*)p;
    else
      return Fmt<DT>::one(*(const uint16_t*)p);
  }
  // Rows are cut into vectors at 16-byte boundaries: the first begins this many
  // elements before the row (4096 rows of 50001 16-bit logits: 79 us, 90 with vectors
  // from the row's own beginning; at 128-byte boundaries 77, but 2000 of a row 15.5
  // against 12.8).
  __device__ static __forceinline__ int32_t before(const char* row) {
    return (int32_t)((uintptr_t)row & 15) / SIZE;
  }
  // STEPS vectors `step` elements apart from element `first` (> -N) of a row on,
  // -infinity before its beginning and past its end.  First all loads of whole
  // vectors; what a row's ends cut is few lanes' business, and in the same loop its
  // shifts would keep every lane waiting (4096 x 50048: 104 us against 70).
  template <int STEPS>
  __device__ static __forceinline__ void load(const char* row, int32_t first, int32_t step, int32_t steps,
                                              int32_t vocab, u32x4 (&v)[STEPS]) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i >= steps) continue;
      const int32_t at = first + i * step;
      v[i] = u32x4{MINUS_INF, MINUS_INF, MINUS_INF, MINUS_INF};
      if (at >= 0 && at + N <= vocab) v[i] = __builtin_nontemporal_load((const u32x4_any*)(row + (int64_t)at * SIZE));
    }
    if (first < 0) v[0] = cut(row, first, vocab);
    const int32_t left = vocab - first;
    int32_t last = left / step;  // the vector that the row's end may cut
    if (left > 0 && left - last * step > 0 && left - last * step < N && last < steps) {
      const u32x4 t = cut(row, first + last * step, vocab);
      asm volatile("" : "+v"(last));  // or the lane masks of all comparisons would be kept
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = i == last ? t[j] : v[i][j];
    }
  }
  // One vector of which only some elements exist.  All its loads travel together (in
  // branches they came one after the other, and every workgroup has such a vector).
  __device__ static __forceinline__ u32x4 cut(const char* row, int32_t at, int32_t vocab) {
    uint32_t e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int32_t in = at + j < 0 ? 0 : at + j < vocab ? at + j : vocab - 1;
      const char* p = row + (int64_t)in * SIZE;
      e[j] = SIZE == 4 ? *(const uint32_t*)p : (uint32_t) * (const uint16_t*)p;
    }
    u32x4 v;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (at + j < 0 || at + j >= vocab) e[j] = SIZE == 4 ? MINUS_INF : MINUS_INF & 0xffffu;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = SIZE == 4 ? e[j] : e[2 * j % N] | e[(2 * j + 1) % N] << 16;
    return v;
  }
  __device__ static __forceinline__ u32x4 load_one(const char* row, int32_t at, int32_t vocab) {
    if (at >= 0 && at + N <= vocab) return *(const u32x4_any*)(row + (int64_t)at * SIZE);
    return cut(row, at, vocab);
  }
};

// A value's place in the order of values as an unsigned integer: NaN above
// +infinity, -0 with +0; 0 is below every value.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  if (order == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order);
}
// a key: its value's order, then the lower index first
__device__ __forceinline__ u64 key_of(uint32_t order, int32_t index) {
  return (u64)order << 32 | (0xffffffffu - (uint32_t)index);
}

struct LogProbArgs {
  const char* logits;
  const int64_t* tokens;
  f32x4* stats;  // [rows, parts]: m, S, the sum of e^(z - m) (z - m)
  u64* keys;     // [rows, parts, top], descending; 0: no value
  float *log_prob, *entropy, *lse, *top_log_prob;
  int64_t* top_index;
  int64_t row_bytes, ignore_index;
  int64_t row_from;                 // first row of the launch
  int32_t rows, parts, top, vocab;  // rows of the launch
  int32_t steps;                    // of a part
  bool cut;                         // into vectors at 16-byte boundaries
};

// ---- the largest values --------------------------------------------------------------------
// Both kernels find the `top` largest keys in two steps.  A bound first: each lane
// has the largest of its own values, and a bound that `top` of the workgroup's lanes
// reach is found bit by bit (ballots), so at least `top` values reach it and, of
// values in no particular place, not many more (256 ln(256 / (256 - top)): 21 for
// 20; with a bound for each wave's 64 lanes four times as many, and 4096 x 50048
// with 20 takes 113 us, 97 so, with 50 211 and 117).  Those that reach it are listed
// in LDS, and each one's place is the number of larger keys.  Where a wave's list
// would be longer (equal values without end) or no bound above -infinity is reached,
// that wave's keys are taken one by one instead, a maximum over its lanes each.
constexpr int kListed = 512;
constexpr uint32_t kOrderMinusInf = 0x007fffffu;

// The largest (or, once they are counted exactly, some) bound that at least `count`
// of some values reach, reached(b) of them b; 0 if there are fewer.  Values of 16
// bits have no bits below LAST.
template <int LAST, class Reached>
__device__ __forceinline__ uint32_t bound_of(Reached&& reached, int count) {
  uint32_t bound = 0;
  for (int bit = 31; bit >= LAST; --bit) {
    const uint32_t b = bound | 1u << bit;
    const int n = reached(b);
    if (n >= count) bound = b;
    if (n == count) break;
  }
  return bound;
}

// Appends the keys of `lanes` to a wave's list; *count goes on past its end.
template <class Key>
__device__ __forceinline__ void append(u64* list, int* count, u64 lanes, Key&& key) {
  const int at = *count + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32),
                                                         __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u));
  if ((lanes >> (threadIdx.x & 63) & 1) && at < kListed) list[at] = key();
  *count += __popcll(lanes);
}

// The number of keys above `key` in a list.
__device__ __forceinline__ int above(const u64* list, int count, u64 key) {
  int n = 0;
#pragma unroll 8
  for (int i = 0; i < count; ++i) n += list[i] > key;
  return n;
}

// ... among the first `count` lanes' keys, the others' being 0: through the scalar
// registers, 8 at a time (one by one, 50 keys take 2 us: each waits for the last).
__device__ __forceinline__ int above_in_lanes(int count, u64 key) {
  const int lo = (int)(uint32_t)key, hi = (int)(uint32_t)(key >> 32);
  int n = 0;
  for (int i = 0; i < count; i += 8) {
    u64 other[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      other[j] = (u64)(uint32_t)__builtin_amdgcn_readlane(hi, i + j) << 32 |
                 (uint32_t)__builtin_amdgcn_readlane(lo, i + j);
#pragma unroll
    for (int j = 0; j < 8; ++j) n += other[j] > key;
  }
  return n;
}

// What a row's sums give.
__device__ __forceinline__ void store_row(const LogProbArgs& a, int64_t row, int64_t token, int dtype, float m, float s,
                                          float t) {
  const bool none = m == -__builtin_inff();
  const float log_s = logf(s), lse = none ? m : m + log_s;
  float z = __builtin_nanf("");
  if (token >= 0 && token < a.vocab) {
    const char* p = a.logits + row * a.row_bytes;
    z = dtype == HPRMS_DTYPE_FP32   ? ((const float*)p)[token]
        : dtype == HPRMS_DTYPE_BF16 ? Fmt<HPRMS_DTYPE_BF16>::one(((const uint16_t*)p)[token])
                                    : Fmt<HPRMS_DTYPE_FP16>::one(((const uint16_t*)p)[token]);
  }
  a.log_prob[row] = none ? z : z - lse;
  a.entropy[row] = none ? 0.0f : log_s - t / s;
  a.lse[row] = lse;
}

__device__ __forceinline__ void store_top(const LogProbArgs& a, int64_t row, int place, u64 key, float lse) {
  const float v = value_of((uint32_t)(key >> 32));
  a.top_log_prob[row * a.top + place] = lse == -__builtin_inff() ? v : v - lse;
  a.top_index[row * a.top + place] = 0xffffffffu - (uint32_t)key;
}

// Parts' maxima and sums, as one.
struct Sums {
  float m, s, t;
  __device__ __forceinline__ void add(float om, float os, float ot) {
    if (om == -__builtin_inff()) return;  // nothing there
    const float top = __builtin_elementwise_maximum(m, om);
    const float d = m == -__builtin_inff() ? kLowest : __builtin_elementwise_maximum(m - top, kLowest);
    const float od = __builtin_elementwise_maximum(om - top, kLowest), f = expf(d), of = expf(od);
    t = f * (t + s * d) + of * (ot + os * od);
    s = f * s + of * os;
    m = top;
  }
};

// 5 workgroups a CU, where 16 vectors a lane take 64 of the 96 registers (with 4
// 4096 x 50048 and 5 alternatives takes 87 us, 82 so; with 8 vectors a lane and 8
// workgroups 87).
template <int DT, bool TOP, int STEPS>
__global__ __launch_bounds__(256, STEPS > 4 ? 5 : 8) void log_probs_part_kernel(LogProbArgs a) {
  using L = Logits<DT>;
  __shared__ u64 lists[TOP ? 4 : 1][TOP ? kListed : 1];
  __shared__ f32x4 stats[4];
  __shared__ uint32_t tops[TOP ? 256 : 1];
  __shared__ int counts[4];
  __shared__ float row_lse;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t here = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int64_t row = a.row_from + here;
  const int64_t token = a.tokens[row];
  if (token == a.ignore_index) {
    if (a.parts == 1) {
      if (threadIdx.x == 0) a.log_prob[row] = a.entropy[row] = a.lse[row] = 0.0f;
      if (TOP && threadIdx.x < a.top) {
        a.top_log_prob[row * a.top + threadIdx.x] = 0.0f;
        a.top_index[row * a.top + threadIdx.x] = -1;
      }
    }
    return;
  }
  const char* z = a.logits + row * a.row_bytes;
  const int32_t first = part * (a.steps * 256 * L::N) + threadIdx.x * L::N - (a.cut ? L::before(z) : 0);
  u32x4 v[STEPS];
  L::template load<STEPS>(z, first, 256 * L::N, a.steps, a.vocab, v);
  float top[STEPS], m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i >= a.steps) continue;
    top[i] = L::get(v[i], 0);
#pragma unroll
    for (int j = 1; j < L::N; ++j) top[i] = __builtin_elementwise_maximum(top[i], L::get(v[i], j));
    m = __builtin_elementwise_maximum(m, top[i]);
  }
  const float lane_top = m;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, d));
  // unpacked again below: the compiler would keep the 128 values otherwise
#pragma unroll
  for (int i = 0; i < STEPS; ++i) packed_again(v[i]);
  const float shift = m == -__builtin_inff() ? 0.0f : m;  // nothing but -infinity: every exponential is 0
  float s = 0.0f, t = 0.0f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i >= a.steps) continue;
#pragma unroll
    for (int j = 0; j < L::N; ++j) {
      const float x = __builtin_elementwise_maximum((L::get(v[i], j) - shift) * kLog2e, kLowest);
      const float e = __builtin_amdgcn_exp2f(x);
      s += e;
      t += e * x;
    }
  }
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  if (lane == 0) stats[wave] = f32x4{m, s, t * kLn2, 0.0f};
  if constexpr (TOP) tops[threadIdx.x] = first < a.vocab ? order_of(lane_top) : 0u;
  __syncthreads();
  if (wave == 0) {
    Sums sums = {stats[0][0], stats[0][1], stats[0][2]};
    for (int w = 1; w < 4; ++w) sums.add(stats[w][0], stats[w][1], stats[w][2]);
    if (a.parts == 1) {
      if (lane == 0) store_row(a, row, token, DT, sums.m, sums.s, sums.t);
      if (TOP && lane == 0) row_lse = sums.m == -__builtin_inff() ? sums.m : sums.m + logf(sums.s);
    } else if (lane == 0) {
      a.stats[(int64_t)here * a.parts + part] = f32x4{sums.m, sums.s, sums.t, 0.0f};
    }
  }
  if constexpr (TOP) {
    u64* list = lists[wave];
    int count = 0;
    uint32_t reach[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) reach[w] = tops[w * 64 + lane];
    const uint32_t bound = bound_of<L::LAST_BIT>(
        [&](uint32_t b) {
          int n = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) n += __popcll(__ballot(reach[w] >= b));
          return n;
        },
        a.top);
    const float least = value_of(bound);
    // (below, what a bound at -infinity would let pass: elements past the row's end)
    bool listed = bound > kOrderMinusInf && bound <= 0xff800000u;
    if (listed) {
      uint32_t hits = 0;  // the lane's steps with a value that reaches it
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        if (i < a.steps && !(top[i] < least)) hits |= 1u << i;
      // Each lane's first such vector, picked from its registers by selects: 80
      // instructions, where a load of it again waits (32 rows x 131072, top 20: 17.8 us
      // for both kernels, 17.0 so).
      while (__ballot(hits != 0) != 0) {
        const int step = hits ? __builtin_ctz(hits) : STEPS;
        const int32_t index = first + step * 256 * L::N;
        u32x4 w = {L::MINUS_INF, L::MINUS_INF, L::MINUS_INF, L::MINUS_INF};
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = i == step ? v[i][j] : w[j];
        hits &= hits - 1;
#pragma unroll
        for (int j = 0; j < L::N; ++j) {
          const float f = L::get(w, j);
          const u64 lanes = __ballot(!(f < least));
          if (lanes != 0) append(list, &count, lanes, [&] { return key_of(order_of(f), index + j); });
        }
        if (count > kListed) break;
      }
      listed = count <= kListed;
    }
    if (!listed) {
      uint32_t order[STEPS];  // of each vector's largest value that is left
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        order[i] = i < a.steps && first + i * 256 * L::N < a.vocab ? order_of(top[i]) : 0u;
      u64 last_key = 0;
      int last_step = -1;
      for (count = 0; count < a.top; ++count) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) best = __builtin_elementwise_max(best, order[i]);
        const uint32_t most = group_max_u32<64>(best);
        if (most == 0) break;  // nothing is left
        // the first vector that holds it: step, then lane
        int step = STEPS;
#pragma unroll
        for (int i = STEPS - 1; i >= 0; --i)
          if (order[i] == most) step = i;
        const uint32_t place = 0xffffffffu - group_max_u32<64>(0xffffffffu - (uint32_t)(step * 64 + lane));
        step = (int)(place >> 6);
        if ((int)(place & 63) == lane) {
          const int32_t index = first + step * 256 * L::N;
          const u32x4 w = L::load_one(z, index, a.vocab);
          // Left of the vector is what is below the last key taken from it: nothing
          // above `most`, and of values equal to it (taken one after the other, as a
          // vector's elements are neighbours) none up to the last one.
          const u64 end = step == last_step ? last_key - 1 : (u64)most << 32 | 0xffffffffu;
          u64 found = 0, next = 0;
#pragma unroll
          for (int j = 0; j < L::N; ++j) {
            const bool in = index + j >= 0 && index + j < a.vocab;
            const u64 key = in ? key_of(order_of(L::get(w, j)), index + j) : 0;
            if (key > end) continue;
            next = key > found ? found : key > next ? key : next;
            found = key > found ? key : found;
          }
          list[count] = found;
          last_key = found;
          last_step = step;
#pragma unroll
          for (int i = 0; i < STEPS; ++i)
            if (i == step) order[i] = (uint32_t)(next >> 32);
        }
      }
    }
    if (lane == 0) counts[wave] = count;
    __syncthreads();
    const float lse = row_lse;
    u64* to = a.keys + ((int64_t)here * a.parts + part) * a.top;
    auto store = [&](int place, u64 key) {
      if (place >= a.top) return;
      if (a.parts == 1)
        store_top(a, row, place, key, lse);
      else
        to[place] = key;
    };
    const int c0 = counts[0], c1 = c0 + counts[1], c2 = c1 + counts[2], all = c2 + counts[3];
    if (all <= 64) {
      if (wave == 0) {
        const int w = lane < c0 ? 0 : lane < c1 ? 1 : lane < c2 ? 2 : 3;
        const int at = lane - (w == 0 ? 0 : w == 1 ? c0 : w == 2 ? c1 : c2);
        const u64 key = lane < all ? lists[w][at] : 0;
        const int place = above_in_lanes(all, key);
        if (lane < all) store(place, key);
      }
    } else {
      for (int i = lane; i < count; i += 64) {
        const u64 key = list[i];
        int place = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) place += above(lists[w], counts[w], key);
        store(place, key);
      }
    }
    // a part of fewer values than alternatives
    if (a.parts > 1 && (int)threadIdx.x >= all && (int)threadIdx.x < a.top) to[threadIdx.x] = 0;
  }
}

// Joins the parts of a row, one wave each.
__global__ __launch_bounds__(256) void log_probs_join_kernel(LogProbArgs a, int dtype) {
  __shared__ u64 lists[4][kListed];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t here = blockIdx.x * 4 + wave;
  if (here >= a.rows) return;
  const int64_t row = a.row_from + here;
  const int64_t token = a.tokens[row];
  if (token == a.ignore_index) {
    if (lane == 0) a.log_prob[row] = a.entropy[row] = a.lse[row] = 0.0f;
    if (lane < a.top) {
      a.top_log_prob[row * a.top + lane] = 0.0f;
      a.top_index[row * a.top + lane] = -1;
    }
    return;
  }
  // lane l has part l, and its list, in descending order
  const bool mine = lane < a.parts;
  const u64* keys = a.keys + ((int64_t)here * a.parts + (mine ? lane : 0)) * a.top;
  constexpr int U = 4;  // loads on their way at once
  u64 key[U];
#pragma unroll
  for (int u = 0; u < U; ++u) key[u] = mine && u < a.top ? keys[u] : 0;
  const f32x4 p = mine ? a.stats[(int64_t)here * a.parts + lane] : f32x4{-__builtin_inff(), 0.0f, 0.0f, 0.0f};
  float m = p[0];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, d));
  float s = 0.0f, t = 0.0f;
  if (p[0] != -__builtin_inff()) {
    const float d = __builtin_elementwise_maximum(p[0] - m, kLowest), f = expf(d);
    s = f * p[1];
    t = f * (p[2] + p[1] * d);
  }
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  if (lane == 0) store_row(a, row, token, dtype, m, s, t);
  if (a.top == 0) return;
  const float lse = m == -__builtin_inff() ? m : m + logf(s);
  // a bound from the lists' r-th keys: r of them each in enough lists
  const int r = (a.top + a.parts - 1) / a.parts, enough = (a.top + r - 1) / r;
  uint32_t reach = mine ? (uint32_t)(keys[r - 1] >> 32) : 0u;
  const uint32_t bound = bound_of<0>([&](uint32_t b) { return __popcll(__ballot(reach >= b)); }, enough);
  u64* list = lists[wave];
  int count = 0;
  bool more = mine;
  for (int n = 0; n < a.top; n += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      more = more && key[u] != 0 && (uint32_t)(key[u] >> 32) >= bound;
      const u64 lanes = __ballot(more);
      if (lanes != 0) append(list, &count, lanes, [&] { return key[u]; });
    }
    if (count > kListed || __ballot(more) == 0) break;
#pragma unroll
    for (int u = 0; u < U; ++u) key[u] = more && n + U + u < a.top ? keys[n + U + u] : 0;
  }
  if (count <= kListed) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the lanes' writes, in order within the wave
    if (count <= 64) {
      const u64 one = lane < count ? list[lane] : 0;
      const int place = above_in_lanes(count, one);
      if (lane < count && place < a.top) store_top(a, row, place, one, lse);
      return;
    }
    for (int i = lane; i < count; i += 64) {
      const int place = above(list, count, list[i]);
      if (place < a.top) store_top(a, row, place, list[i], lse);
    }
    return;
  }
  u64 head = mine ? keys[0] : 0;
  int used = 0;
  for (int n = 0; n < a.top; ++n) {
    const uint32_t hi = group_max_u32<64>((uint32_t)(head >> 32));
    const uint32_t lo = group_max_u32<64>((uint32_t)(head >> 32) == hi ? (uint32_t)head : 0u);
    const u64 most = (u64)hi << 32 | lo;
    if (lane == 0) store_top(a, row, n, most, lse);
    if (head == most) head = ++used < a.top ? keys[used] : 0;
  }
}

// ---- gradient ---------------------------------------------------------------------------
struct LogProbGradArgs {
  char* dlogits;
  const char* logits;
  const int64_t* tokens;
  const float *dlog_prob, *dentropy, *lse, *entropy;  // dentropy and entropy may be null
  int64_t dlogits_bytes, logits_bytes, ignore_index, row_from;
  int32_t parts, vocab;
};

// One workgroup: 4 steps of 256 vectors of one row.
constexpr int kGradSteps = 4;

template <int DT>
__global__ __launch_bounds__(256) void log_probs_grad_kernel(LogProbGradArgs a) {
  using L = Logits<DT>;
  const int64_t row = a.row_from + blockIdx.x / a.parts;
  const char* z = a.logits + row * a.logits_bytes;
  char* to = a.dlogits + row * a.dlogits_bytes;
  const int32_t first =
      (int32_t)(blockIdx.x % a.parts) * (256 * kGradSteps * L::N) + threadIdx.x * L::N - L::before(to);
  const int64_t token = a.tokens[row];
  const bool ignored = token == a.ignore_index;
  const float lse = a.lse[row];
  const bool none = ignored || lse == -__builtin_inff();  // no probabilities: zeros
  const float g = token >= 0 && token < a.vocab ? a.dlog_prob[row] : __builtin_nanf("");
  const float gh = a.dentropy ? a.dentropy[row] : 0.0f, entropy = a.dentropy ? a.entropy[row] : 0.0f;
  const float by = -g - gh * entropy, per = -gh * kLn2;  // dz = p * (by + per * log2 p) + [v == token] g
  u32x4 v[kGradSteps];
  if (!ignored) L::template load<kGradSteps>(z, first, 256 * L::N, kGradSteps, a.vocab, v);
#pragma unroll
  for (int i = 0; i < kGradSteps; ++i) {
    const int32_t index = first + i * 256 * L::N;
    if (index >= a.vocab) continue;
    float d[L::N];
#pragma unroll
    for (int j = 0; j < L::N; ++j) {
      d[j] = 0.0f;
      if (!none) {
        const float x = __builtin_elementwise_maximum((L::get(v[i], j) - lse) * kLog2e, kLowest);
        d[j] = __builtin_amdgcn_exp2f(x) * (by + per * x);
        if (index + j == token) d[j] += g;
      }
    }
    u32x4 o;
    if constexpr (DT == HPRMS_DTYPE_FP32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __float_as_uint(d[j]);
    } else {
      o = pack8<DT>(d);
    }
    if (index >= 0 && index + L::N <= a.vocab) {
      __builtin_nontemporal_store(o, (u32x4_any*)(to + index * L::SIZE));
    } else {
#pragma unroll
      for (int j = 0; j < L::N; ++j)
        if (index + j >= 0 && index + j < a.vocab) {
          if constexpr (DT == HPRMS_DTYPE_FP32)
            *(uint32_t*)(to + (index + j) * 4) = o[j];
          else
            *(uint16_t*)(to + (index + j) * 2) = (uint16_t)(o[j / 2] >> (16 * (j & 1)));
        }
    }
  }
}

// ---- host ------------------------------------------------------------------------------
constexpr int64_t kMaxRows = int64_t(1) << 31;
constexpr int64_t kMaxVocab = int64_t(1) << 20;
constexpr int64_t kMaxPartials = int64_t(1) << 26;  // bytes of partial results: more rows take more launches

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t size_of(int dtype) { return dtype == HPRMS_DTYPE_FP32 ? 4 : 2; }

// A row's bytes, with what its first vector may hold before it.
int64_t row_bytes_of(int64_t vocab, int dtype, bool cut) {
  return vocab * size_of(dtype) + (cut ? 16 - size_of(dtype) : 0);
}

// Parts of a row: as few as hold it, or, for few rows, so many that two workgroups
// a CU have some, of 2 steps at least.  In batch-invariant mode always the fewest:
// other parts sum a row's exponentials in another order, which shows in last bits.
// For the same reason rows are cut from their own beginning there, wherever they lie
// (plan_of): vectors at 16-byte boundaries would be others for each row of an odd
// stride, and the bytes before the first can take a part more (4096 x 50001 bf16, 5
// alternatives: 94 us so, 84 cut at the boundaries).
int64_t parts_of(int64_t rows, int64_t bytes, bool invariant) {
  const int64_t least = (bytes + kPartBytes - 1) / kPartBytes, most = (bytes + 2 * kStepBytes - 1) / (2 * kStepBytes);
  int64_t parts = least;
  if (!invariant && rows > 0) parts = (2 * (int64_t)current_cus() + rows - 1) / rows;
  if (parts > most) parts = most;
  if (parts > kMaxParts) parts = kMaxParts;
  return parts < least ? least : parts;
}

struct Plan {
  int64_t parts, steps, rows_at, keys, total;  // rows of a launch; bytes
  bool cut;
};
// `aligned`: every row begins at a 16-byte boundary
Plan plan_of(int64_t rows, int64_t vocab, int64_t top, int dtype, bool invariant, bool aligned) {
  Plan p;
  // (the largest vocabularies fill the most parts there can be)
  p.cut = !aligned && !invariant && row_bytes_of(vocab, dtype, true) <= kMaxParts * kPartBytes;
  const int64_t bytes = row_bytes_of(vocab, dtype, p.cut);
  p.parts = parts_of(rows, bytes, invariant);
  p.steps = (bytes + p.parts * kStepBytes - 1) / (p.parts * kStepBytes);
  const int64_t row = p.parts * (16 + 8 * top);
  p.rows_at = kMaxPartials / row;
  if (p.rows_at > rows) p.rows_at = rows;
  p.keys = round_up(p.rows_at * p.parts * 16, 256);
  p.total = p.parts == 1 ? 0 : p.keys + p.rows_at * p.parts * top * 8;
  return p;
}

int check_sizes(int64_t rows, int64_t vocab, int64_t top, int dtype) {
  if (dtype != HPRMS_DTYPE_BF16 && dtype != HPRMS_DTYPE_FP16 && dtype != HPRMS_DTYPE_FP32)
    return fail(HPRMS_E_INVALID, "dtype must be an hprms_dtype (got %d)", dtype);
  if (rows < 0) return fail(HPRMS_E_INVALID, "rows must be >= 0 (got %lld)", (long long)rows);
  if (vocab < 1) return fail(HPRMS_E_INVALID, "vocab must be >= 1 (got %lld)", (long long)vocab);
  if (rows >= kMaxRows || vocab > kMaxVocab)
    return fail(HPRMS_E_RANGE, "rows must be below 2^31 and vocab at most 2^20 (got %lld, %lld)", (long long)rows,
                (long long)vocab);
  if (top < 0 || top > kMaxTop || top > vocab)
    return fail(HPRMS_E_INVALID, "top must be from 0 to %d and at most vocab (got %lld)", kMaxTop, (long long)top);
  return HPRMS_OK;
}

bool aligned_to(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <int DT, bool TOP>
void launch_parts(const LogProbArgs& a, dim3 grid, dim3 block, hipStream_t stream) {
  if (a.steps <= 4)
    log_probs_part_kernel<DT, TOP, 4><<<grid, block, 0, stream>>>(a);
  else
    log_probs_part_kernel<DT, TOP, kSteps><<<grid, block, 0, stream>>>(a);
}

template <int DT>
int run_forward(LogProbArgs a, const Plan& p, int64_t rows, hipStream_t stream) {
  for (int64_t from = 0; from < rows; from += p.rows_at) {
    a.row_from = from;
    a.rows = (int32_t)(rows - from < p.rows_at ? rows - from : p.rows_at);
    const dim3 grid((unsigned)(a.rows * p.parts)), block(256);
    if (a.top > 0)
      launch_parts<DT, true>(a, grid, block, stream);
    else
      launch_parts<DT, false>(a, grid, block, stream);
    if (p.parts > 1) log_probs_join_kernel<<<dim3((unsigned)((a.rows + 3) / 4)), block, 0, stream>>>(a, DT);
  }
  return check_launch("log probability kernel");
}

template <int DT>
int run_backward(LogProbGradArgs a, int64_t rows, hipStream_t stream) {
  const int64_t span = 256 * kGradSteps * Logits<DT>::N;
  a.parts = (int32_t)((a.vocab + Logits<DT>::N - 1 + span - 1) / span);
  const int64_t rows_at = (int64_t(1) << 23) / a.parts;  // a launch holds fewer than 2^32 work-items
  for (int64_t from = 0; from < rows; from += rows_at) {
    a.row_from = from;
    const int64_t here = rows - from < rows_at ? rows - from : rows_at;
    log_probs_grad_kernel<DT><<<dim3((unsigned)(here * a.parts)), dim3(256), 0, stream>>>(a);
  }
  return check_launch("log probability gradient kernel");
}

}  // namespace
}  // namespace hprms

using namespace hprms;

extern "C" {

int64_t hprms_token_log_probs_workspace(int64_t rows, int64_t vocab, int64_t top, int dtype) {
  const int rc = check_sizes(rows, vocab, top, dtype);
  if (rc != HPRMS_OK || rows == 0) return rc;
  // enough for either mode, which may change between the query and the call, and wherever the rows begin
  int64_t most = 0;
  for (int i = 0; i < 4; ++i) {
    const int64_t n = plan_of(rows, vocab, top, dtype, i & 1, i & 2).total;
    if (n > most) most = n;
  }
  return most;
}

int hprms_token_log_probs(float* log_prob, float* entropy, float* lse, float* top_log_prob, int64_t* top_index,
                          const void* logits, const int64_t* tokens, void* workspace, int64_t workspace_size,
                          int64_t rows, int64_t vocab, int64_t top, int64_t logits_row_stride, int64_t ignore_index,
                          int dtype, hipStream_t stream) {
  const int rc = check_sizes(rows, vocab, top, dtype);
  if (rc != HPRMS_OK) return rc;
  if (logits_row_stride < vocab) return fail(HPRMS_E_INVALID, "row strides must be >= vocab");
  const int64_t size = size_of(dtype);
  if (!extent_ok(rows, logits_row_stride, size, vocab))
    return fail(HPRMS_E_RANGE, "%lld rows at this row stride span more than 2^56 bytes", (long long)rows);
  if (rows == 0) return HPRMS_OK;
  if (!log_prob || !entropy || !lse || !logits || !tokens || (top > 0 && (!top_log_prob || !top_index)))
    return fail(HPRMS_E_INVALID, "null tensor pointer");
  if (!aligned_to(log_prob, 4) || !aligned_to(entropy, 4) || !aligned_to(lse, 4) || !aligned_to(logits, size) ||
      !aligned_to(tokens, 8) || (top > 0 && (!aligned_to(top_log_prob, 4) || !aligned_to(top_index, 8))))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  const Plan p = plan_of(rows, vocab, top, dtype, hprms_batch_invariant() != 0,
                         aligned_to(logits, 16) && (rows == 1 || logits_row_stride * size % 16 == 0));
  if (p.total > 0 && (!workspace || workspace_size < p.total || !aligned_to(workspace, 16)))
    return fail(HPRMS_E_INVALID, "the workspace must hold %lld bytes, 16-byte aligned (got %lld)", (long long)p.total,
                (long long)workspace_size);
  LogProbArgs a = {};
  a.logits = (const char*)logits;
  a.tokens = tokens;
  a.stats = (f32x4*)workspace;
  a.keys = (u64*)((char*)workspace + p.keys);
  a.log_prob = log_prob;
  a.entropy = entropy;
  a.lse = lse;
  a.top_log_prob = top_log_prob;
  a.top_index = top_index;
  a.row_bytes = logits_row_stride * size;
  a.vocab = (int32_t)vocab;
  a.ignore_index = ignore_index;
  a.parts = (int32_t)p.parts;
  a.steps = (int32_t)p.steps;
  a.cut = p.cut;
  a.top = (int32_t)top;
  return dtype == HPRMS_DTYPE_FP32   ? run_forward<HPRMS_DTYPE_FP32>(a, p, rows, stream)
         : dtype == HPRMS_DTYPE_BF16 ? run_forward<HPRMS_DTYPE_BF16>(a, p, rows, stream)
                                     : run_forward<HPRMS_DTYPE_FP16>(a, p, rows, stream);
}

int hprms_token_log_probs_backward(void* dlogits, const float* dlog_prob, const float* dentropy, const void* logits,
                                   const int64_t* tokens, const float* lse, const float* entropy, int64_t rows,
                                   int64_t vocab, int64_t dlogits_row_stride, int64_t logits_row_stride,
                                   int64_t ignore_index, int dtype, hipStream_t stream) {
  const int rc = check_sizes(rows, vocab, 0, dtype);
  if (rc != HPRMS_OK) return rc;
  if (dlogits_row_stride < vocab || logits_row_stride < vocab)
    return fail(HPRMS_E_INVALID, "row strides must be >= vocab");
  const int64_t size = size_of(dtype);
  if (!extent_ok(rows, dlogits_row_stride, size, vocab) || !extent_ok(rows, logits_row_stride, size, vocab))
    return fail(HPRMS_E_RANGE, "%lld rows at these row strides span more than 2^56 bytes", (long long)rows);
  if (rows == 0) return HPRMS_OK;
  if (!dlogits || !dlog_prob || !logits || !tokens || !lse || (dentropy && !entropy))
    return fail(HPRMS_E_INVALID, "null tensor pointer");
  if (!aligned_to(dlogits, size) || !aligned_to(logits, size) || !aligned_to(dlog_prob, 4) || !aligned_to(lse, 4) ||
      !aligned_to(dentropy, 4) || (dentropy && !aligned_to(entropy, 4)) || !aligned_to(tokens, 8))
    return fail(HPRMS_E_INVALID, "tensors must be aligned to their elements");
  if (dlogits == logits && rows > 1 && dlogits_row_stride != logits_row_stride)
    return fail(HPRMS_E_INVALID, "an in-place alias needs equal row strides");
  LogProbGradArgs a = {};
  a.dlogits = (char*)dlogits;
  a.logits = (const char*)logits;
  a.tokens = tokens;
  a.dlog_prob = dlog_prob;
  a.dentropy = dentropy;
  a.lse = lse;
  a.entropy = entropy;
  a.dlogits_bytes = dlogits_row_stride * size;
  a.logits_bytes = logits_row_stride * size;
  a.vocab = (int32_t)vocab;
  a.ignore_index = ignore_index;
  return dtype == HPRMS_DTYPE_FP32   ? run_backward<HPRMS_DTYPE_FP32>(a, rows, stream)
         : dtype == HPRMS_DTYPE_BF16 ? run_backward<HPRMS_DTYPE_BF16>(a, rows, stream)
                                     : run_backward<HPRMS_DTYPE_FP16>(a, rows, stream);
}

}  // extern "C"
