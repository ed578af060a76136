// hprms_log_probs.hip - log probabilities of given tokens under rows of logits, with
// the entropy and the most likely alternatives, and the gradient.
//
//   m = max z;  S = sum e^(z - m);  lse = m + log S;  log_prob = z[token] - lse
//   entropy = log S + (sum e^(z - m) (m - z)) / S      (all terms >= 0)
//   top alternatives: the largest z, equal ones by the lower index, minus lse
//   dz = dlog_prob * ([v == token] - p) - dentropy * p * (log p + entropy)
//
// Forward, first kernel: a wave takes a part of a row, kPartBytes of it, into
// registers at once, 16 bytes a lane and step, and leaves the part's m, S and sum
// of e^(z - m) (z - m) and its `top` largest as sorted keys.  Its loads are all on
// their way before the first is used, waves need no barrier, and the logits are
// read once.  Second kernel: a wave joins a row's parts.  The gradient is one pass
// over the logits, from the forward call's lse and entropy.
#include <hip/hip_runtime.h>

#include "hprms_host.h"
#include "hprms_rows.h"

namespace hprms {
namespace {

typedef unsigned long long u64;

constexpr int kSteps = 16;                 // 16-byte loads of a lane
constexpr int kPartBytes = kSteps * 1024;  // a part: 8192 16-bit or 4096 32-bit logits
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
// exponents of 2 below this give 0; bounds what 0 is multiplied with at -infinity
constexpr float kLowest = -200.0f;

template <int DT>
struct Logits {
  static constexpr int N = DT == HPRMS_DTYPE_FP32 ? 4 : 8;  // of a vector
  static constexpr int SIZE = DT == HPRMS_DTYPE_FP32 ? 4 : 2;
  static constexpr int PART = kPartBytes / SIZE;
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
  // the vector at element i of a row, -infinity past the row's end
  __device__ static __forceinline__ u32x4 load(const char* row, int32_t i, int32_t vocab) {
    if (i + N <= vocab) return __builtin_nontemporal_load((const u32x4_any*)(row + i * SIZE));
    u32x4 v = {MINUS_INF, MINUS_INF, MINUS_INF, MINUS_INF};
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j < vocab) {
        if constexpr (DT == HPRMS_DTYPE_FP32)
          v[j] = *(const uint32_t*)(row + (i + j) * 4);
        else if (j & 1)
          v[j / 2] = (v[j / 2] & 0xffffu) | (uint32_t) * (const uint16_t*)(row + (i + j) * 2) << 16;
        else
          v[j / 2] = (v[j / 2] & 0xffff0000u) | *(const uint16_t*)(row + (i + j) * 2);
      }
    return v;
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
};

template <int DT, bool TOP>
__global__ __launch_bounds__(256, 4) void log_probs_part_kernel(LogProbArgs a) {
  using L = Logits<DT>;
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t here = (int32_t)(at / a.parts), part = (int32_t)(at % a.parts);
  if (here >= a.rows) return;
  const int64_t row = a.row_from + here;
  if (a.tokens[row] == a.ignore_index) return;
  const char* z = a.logits + row * a.row_bytes;
  const int32_t first = part * L::PART + lane * L::N;
  u32x4 v[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) v[i] = L::load(z, first + i * 64 * L::N, a.vocab);
  float top[kSteps], m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    top[i] = L::get(v[i], 0);
#pragma unroll
    for (int j = 1; j < L::N; ++j) top[i] = __builtin_elementwise_maximum(top[i], L::get(v[i], j));
    m = __builtin_elementwise_maximum(m, top[i]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, d));
  // unpacked again below: the compiler would keep the 128 values otherwise
#pragma unroll
  for (int i = 0; i < kSteps; ++i) asm volatile("" : "+v"(v[i]));
  const float shift = m == -__builtin_inff() ? 0.0f : m;  // nothing but -infinity: every exponential is 0
  float s = 0.0f, t = 0.0f;
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
#pragma unroll
    for (int j = 0; j < L::N; ++j) {
      const float x = __builtin_elementwise_maximum((L::get(v[i], j) - shift) * kLog2e, kLowest);
      const float e = __builtin_amdgcn_exp2f(x);
      s += e;
      t += e * x;
    }
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  if (lane == 0) a.stats[(int64_t)here * a.parts + part] = f32x4{m, s, t * kLn2, 0.0f};
  if constexpr (TOP) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) asm volatile("" : "+v"(v[i]));
    uint32_t order[kSteps];     // of each vector's largest value that is left
    uint32_t gone[kSteps / 4];  // what is taken, 8 bits a vector
#pragma unroll
    for (int i = 0; i < kSteps; ++i) order[i] = first + i * 64 * L::N < a.vocab ? order_of(top[i]) : 0u;
#pragma unroll
    for (int i = 0; i < kSteps / 4; ++i) gone[i] = 0;
    u64* to = a.keys + ((int64_t)here * a.parts + part) * a.top;
    for (int n = 0; n < a.top; ++n) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) best = __builtin_elementwise_max(best, order[i]);
      const uint32_t most = group_max_u32<64>(best);
      if (most == 0) {  // fewer values than alternatives
        if (lane == 0)
          for (int i = n; i < a.top; ++i) to[i] = 0;
        break;
      }
      // the first vector that holds it: step, then lane
      int step = kSteps;
#pragma unroll
      for (int i = kSteps - 1; i >= 0; --i)
        if (order[i] == most) step = i;
      const uint32_t place = 0xffffffffu - group_max_u32<64>(0xffffffffu - (uint32_t)(step * 64 + lane));
      const int s0 = (int)(place >> 6);
      const bool mine = (int)(place & 63) == lane;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (i != s0) continue;  // the same for all lanes
        const int32_t index = first + i * 64 * L::N;
        // opaque: the orders of all 128 values would be kept over the loop otherwise
        u32x4 w = v[i];
        uint32_t taken = gone[i / 4] >> (8 * (i & 3));
        int valid = a.vocab - index;
        asm volatile("" : "+v"(w), "+v"(taken), "+v"(valid));
        uint32_t left = 0;
        int found = -1;
#pragma unroll
        for (int j = 0; j < L::N; ++j) {
          uint32_t o = order_of(L::get(w, j));
          if (taken & (1u << j) || j >= valid) o = 0;
          if (o == most && found < 0)
            found = j;
          else
            left = __builtin_elementwise_max(left, o);
        }
        if (mine) {
          to[n] = key_of(most, index + found);
          gone[i / 4] |= 1u << (8 * (i & 3) + found);
          order[i] = left;
        }
      }
    }
  }
}

// Joins the parts of a row, one wave each.
__global__ __launch_bounds__(256) void log_probs_join_kernel(LogProbArgs a, int dtype) {
  const int lane = threadIdx.x & 63;
  const int32_t here = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (here >= a.rows) return;
  const int64_t row = a.row_from + here;
  const int64_t token = a.tokens[row];
  float* top_log_prob = a.top_log_prob + row * a.top;
  int64_t* top_index = a.top_index + row * a.top;
  if (token == a.ignore_index) {
    if (lane == 0) a.log_prob[row] = a.entropy[row] = a.lse[row] = 0.0f;
    if (lane < a.top) {
      top_log_prob[lane] = 0.0f;
      top_index[lane] = -1;
    }
    return;
  }
  const f32x4* stats = a.stats + (int64_t)here * a.parts;
  float m = -__builtin_inff();
  for (int i = lane; i < a.parts; i += 64) m = __builtin_elementwise_maximum(m, stats[i][0]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, d));
  float s = 0.0f, t = 0.0f;
  for (int i = lane; i < a.parts; i += 64) {
    const f32x4 p = stats[i];
    if (p[0] == -__builtin_inff()) continue;  // nothing there
    const float d = __builtin_elementwise_maximum(p[0] - m, kLowest), f = expf(d);
    s += f * p[1];
    t += f * (p[2] + p[1] * d);
  }
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  const bool none = m == -__builtin_inff();
  const float lse = none ? m : m + logf(s);
  if (lane == 0) {
    float z = __builtin_nanf("");
    if (token >= 0 && token < a.vocab) {
      const char* p = a.logits + row * a.row_bytes;
      z = dtype == HPRMS_DTYPE_FP32   ? ((const float*)p)[token]
          : dtype == HPRMS_DTYPE_BF16 ? Fmt<HPRMS_DTYPE_BF16>::one(((const uint16_t*)p)[token])
                                      : Fmt<HPRMS_DTYPE_FP16>::one(((const uint16_t*)p)[token]);
    }
    a.log_prob[row] = none ? z : z - lse;
    a.entropy[row] = none ? 0.0f : logf(s) - t / s;
    a.lse[row] = lse;
  }
  if (a.top == 0) return;
  // lane l has the lists of parts l, l + 64, ...: their first keys that are left
  constexpr int LISTS = 4;
  const u64* keys = a.keys + (int64_t)here * a.parts * a.top;
  u64 head[LISTS];
  int used[LISTS];
#pragma unroll
  for (int i = 0; i < LISTS; ++i) {
    used[i] = 0;
    head[i] = lane + i * 64 < a.parts ? keys[(int64_t)(lane + i * 64) * a.top] : 0;
  }
  u64 mine = 0;  // lane n ends with alternative n
  for (int n = 0; n < a.top; ++n) {
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < LISTS; ++i) best = head[i] > best ? head[i] : best;
    const uint32_t hi = group_max_u32<64>((uint32_t)(best >> 32));
    const uint32_t lo = group_max_u32<64>((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    const u64 most = (u64)hi << 32 | lo;
    if (lane == n) mine = most;
#pragma unroll
    for (int i = 0; i < LISTS; ++i)
      if (head[i] == most) {
        ++used[i];
        head[i] = used[i] < a.top ? keys[(int64_t)(lane + i * 64) * a.top + used[i]] : 0;
      }
  }
  if (lane < a.top) {
    const float v = value_of((uint32_t)(mine >> 32));
    top_log_prob[lane] = none ? v : v - lse;
    top_index[lane] = 0xffffffffu - (uint32_t)mine;
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
  const int32_t first = (int32_t)(blockIdx.x % a.parts) * (256 * kGradSteps * L::N) + threadIdx.x * L::N;
  const char* z = a.logits + row * a.logits_bytes;
  char* to = a.dlogits + row * a.dlogits_bytes;
  const int64_t token = a.tokens[row];
  const bool ignored = token == a.ignore_index;
  const float lse = a.lse[row];
  const bool none = ignored || lse == -__builtin_inff();  // no probabilities: zeros
  const float g = token >= 0 && token < a.vocab ? a.dlog_prob[row] : __builtin_nanf("");
  const float gh = a.dentropy ? a.dentropy[row] : 0.0f, entropy = a.dentropy ? a.entropy[row] : 0.0f;
  const float by = -g - gh * entropy, per = -gh * kLn2;  // dz = p * (by + per * log2 p) + [v == token] g
  u32x4 v[kGradSteps];
  if (!ignored) {
#pragma unroll
    for (int i = 0; i < kGradSteps; ++i) v[i] = L::load(z, first + i * 256 * L::N, a.vocab);
  }
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
    if (index + L::N <= a.vocab) {
      __builtin_nontemporal_store(o, (u32x4_any*)(to + index * L::SIZE));
    } else {
#pragma unroll
      for (int j = 0; j < L::N; ++j)
        if (index + j < a.vocab) {
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
int64_t parts_of(int64_t vocab, int dtype) { return (vocab * size_of(dtype) + kPartBytes - 1) / kPartBytes; }

struct Plan {
  int64_t parts, rows_at, keys, total;  // rows of a launch; bytes
};
Plan plan_of(int64_t rows, int64_t vocab, int64_t top, int dtype) {
  Plan p;
  p.parts = parts_of(vocab, dtype);
  const int64_t row = p.parts * (16 + 8 * top);
  p.rows_at = kMaxPartials / row;
  if (p.rows_at < 1) p.rows_at = 1;
  if (p.rows_at > rows) p.rows_at = rows;
  p.keys = round_up(p.rows_at * p.parts * 16, 256);
  p.total = p.keys + p.rows_at * p.parts * top * 8;
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

template <int DT>
int run_forward(LogProbArgs a, const Plan& p, int64_t rows, hipStream_t stream) {
  for (int64_t from = 0; from < rows; from += p.rows_at) {
    a.row_from = from;
    a.rows = (int32_t)(rows - from < p.rows_at ? rows - from : p.rows_at);
    const dim3 grid((unsigned)((a.rows * p.parts + 3) / 4)), block(256);
    if (a.top > 0)
      log_probs_part_kernel<DT, true><<<grid, block, 0, stream>>>(a);
    else
      log_probs_part_kernel<DT, false><<<grid, block, 0, stream>>>(a);
    log_probs_join_kernel<<<dim3((unsigned)((a.rows + 3) / 4)), block, 0, stream>>>(a, DT);
  }
  return check_launch("log probability kernel");
}

template <int DT>
int run_backward(LogProbGradArgs a, int64_t rows, hipStream_t stream) {
  const int64_t span = 256 * kGradSteps * Logits<DT>::N;
  a.parts = (int32_t)((a.vocab + span - 1) / span);
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
  return rc != HPRMS_OK ? rc : rows == 0 ? 0 : plan_of(rows, vocab, top, dtype).total;
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
  const Plan p = plan_of(rows, vocab, top, dtype);
  if (!workspace || workspace_size < p.total || !aligned_to(workspace, 16))
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
