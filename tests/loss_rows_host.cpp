// loss_pack_kernel (hp_rms_norm_amd/csrc/hprms_loss_rows.h) on the CPU, one
// workgroup after another, its 256 lanes as contexts of one thread.
//
// The waves of a workgroup run in a given order of preference: the first wave
// of that order that does not wait at a barrier runs on, up to the barrier,
// before any other moves.  With an order and its reverse every wave is once as
// far ahead of every other as barriers allow, and a word of LDS that one wave
// overwrites before another has read it shows as a wrong result.
//
//   loss_rows_host <rows> <width> <hidden stride> <ignored, per cent> <seed>
//
// tries both orders, forward and gradient form, and compares everything the
// kernel writes with loops over the rows.
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <algorithm>
#include <vector>

#define __device__
#define __global__
#define __shared__ static
#define __launch_bounds__(n)
#define __forceinline__ inline

struct Dim {
  unsigned x;
};
static Dim threadIdx, blockIdx, gridDim;
struct float2 {
  float x, y;
};

static void wave_op(uint64_t value, uint64_t* all);  // every lane's value, of the wave
static void block_barrier();

static void __syncthreads() { block_barrier(); }
static uint64_t __ballot(bool v) {
  uint64_t all[64], mask = 0;
  wave_op(v, all);
  for (int i = 0; i < 64; ++i) mask |= all[i] << i;
  return mask;
}
template <class T>
static T __shfl_xor(T v, int m) {
  static_assert(sizeof(T) == 4, "one register");
  uint64_t all[64], bits = 0;
  memcpy(&bits, &v, 4);
  wave_op(bits, all);
  memcpy(&v, &all[(threadIdx.x & 63) ^ (unsigned)m], 4);
  return v;
}
static int __popcll(uint64_t v) { return __builtin_popcountll(v); }
static int __float_as_int(float f) {
  int i;
  memcpy(&i, &f, 4);
  return i;
}
static unsigned __float_as_uint(float f) { return (unsigned)__float_as_int(f); }
static float __int_as_float(int i) {
  float f;
  memcpy(&f, &i, 4);
  return f;
}
static float __uint_as_float(unsigned u) { return __int_as_float((int)u); }
using std::max;
using std::min;

#include "hprms_loss_rows.h"

using namespace hprms;

// ---- the lanes -----------------------------------------------------------------------
enum State { kReady, kAtWaveOp, kAtBarrier, kDone };
static const int kLanes = 256, kStack = 64 << 10;
static ucontext_t g_main, g_lane[kLanes];
static std::vector<char> g_stack(kLanes * (size_t)kStack);
static State g_state[kLanes];
static uint64_t g_value[kLanes];
static int g_current;

struct Call {
  bool grad;
  LossArgs a;
  LossMeta* meta;
  int32_t* index;
  uint16_t* packed;
};
static const Call* g_call;

static void yield_as(State s) {
  const int me = g_current;
  g_state[me] = s;
  swapcontext(&g_lane[me], &g_main);
}
static void block_barrier() { yield_as(kAtBarrier); }
static void wave_op(uint64_t value, uint64_t* all) {
  const int me = g_current;
  g_value[me] = value;
  yield_as(kAtWaveOp);
  memcpy(all, &g_value[me & ~63], sizeof(uint64_t) * 64);
  yield_as(kAtWaveOp);  // nobody goes on to its next value before all have read this one
}
static void lane_main() {
  const Call& c = *g_call;
  if (c.grad)
    loss_pack_kernel<true>(c.a, c.meta, c.index, c.packed);
  else
    loss_pack_kernel<false>(c.a, c.meta, c.index, c.packed);
  yield_as(kDone);
}

static void fail(const char* what) {
  printf("FAIL: %s\n", what);
  exit(1);
}

static void run_lane(int lane) {
  g_current = lane;
  threadIdx.x = (unsigned)lane;
  swapcontext(&g_main, &g_lane[lane]);
}

// the wave's lanes up to its next barrier, or the end
static void run_wave(int wave) {
  for (;;) {
    for (int l = wave * 64; l < wave * 64 + 64; ++l)
      if (g_state[l] == kReady) run_lane(l);
    const State s = g_state[wave * 64];
    for (int l = wave * 64; l < wave * 64 + 64; ++l)
      if (g_state[l] != s) fail("the lanes of a wave part ways");
    if (s != kAtWaveOp) return;
    for (int l = wave * 64; l < wave * 64 + 64; ++l) g_state[l] = kReady;
  }
}

static void run_block(const int* order) {
  for (int l = 0; l < kLanes; ++l) {
    getcontext(&g_lane[l]);
    g_lane[l].uc_stack.ss_sp = &g_stack[l * (size_t)kStack];
    g_lane[l].uc_stack.ss_size = kStack;
    g_lane[l].uc_link = &g_main;
    makecontext(&g_lane[l], lane_main, 0);
    g_state[l] = kReady;
  }
  for (;;) {
    for (int i = 0; i < 4; ++i)
      if (g_state[order[i] * 64] == kReady) run_wave(order[i]);
    int waiting = 0;
    for (int w = 0; w < 4; ++w) waiting += g_state[w * 64] == kAtBarrier;
    if (waiting == 0) return;
    if (waiting != 4) fail("not every wave reaches a barrier");
    for (int l = 0; l < kLanes; ++l) g_state[l] = kReady;
  }
}

// ---- the call ------------------------------------------------------------------------
static uint32_t g_seed;
static uint32_t next_random() { return (g_seed = g_seed * 1664525u + 1013904223u) >> 8; }

template <class T>
static void same(const std::vector<T>& got, const std::vector<T>& want, const char* what) {
  if (memcmp(got.data(), want.data(), sizeof(T) * got.size()) != 0) fail(what);
}

int main(int argc, char** argv) {
  if (argc != 6) return 2;
  const int rows = atoi(argv[1]), width = atoi(argv[2]), stride = atoi(argv[3]), ignored = atoi(argv[4]);
  g_seed = (uint32_t)atoi(argv[5]);
  const int packed_width = (width + 63) / 64 * 64;
  // what a wrong place may reach: a workgroup's 256 rows more, before and behind
  const int slack = 512;
  std::vector<uint16_t> hidden((size_t)rows * stride);
  std::vector<int64_t> target(rows);
  std::vector<float> dloss(rows);
  for (auto& v : hidden) v = (uint16_t)next_random();
  for (auto& t : target) t = (int)(next_random() % 100) < ignored ? -100 : next_random() % 1000;
  for (auto& g : dloss) g = (float)(next_random() % 1000) / 64.0f;
  const int orders[2][4] = {{0, 1, 2, 3}, {3, 2, 1, 0}};
  for (const int* order : orders) {
    for (int grad = 0; grad < 2; ++grad) {
      const size_t n = rows + 2 * slack;
      std::vector<int32_t> index(n, -7), want_index(n, -7);
      std::vector<uint16_t> packed(n * packed_width, 0x5555), want_packed(packed);
      std::vector<float> loss(rows, 9.0f), lse(rows, 9.0f), want_loss(loss);
      std::vector<uint16_t> dhidden((size_t)rows * stride, 0x7777), want_dhidden(dhidden);
      LossMeta meta = {-1, -1.0f, -1.0f, 0};
      Call c = {};
      c.grad = grad;
      c.a.hidden = hidden.data();
      c.a.target = target.data();
      c.a.dloss = dloss.data();
      c.a.hidden_stride = c.a.dhidden_stride = stride;
      c.a.ignore_index = -100;
      c.a.packed_width = packed_width;
      c.a.rows = rows;
      c.a.width = width;
      c.a.loss = loss.data();
      c.a.lse = lse.data();
      c.a.dhidden = dhidden.data();
      c.a.pack_rows = (rows + 511) / 512;
      c.meta = &meta;
      c.index = index.data() + slack;
      c.packed = packed.data() + (size_t)slack * packed_width;
      g_call = &c;
      const int groups = (rows + c.a.pack_rows - 1) / c.a.pack_rows;
      gridDim.x = groups + grad;
      for (blockIdx.x = 0; blockIdx.x < gridDim.x; ++blockIdx.x) run_block(order);

      int count = 0;
      float top = 0.0f;
      for (int r = 0; r < rows; ++r) {
        if (target[r] != -100) {
          want_index[slack + count] = r;
          uint16_t* to = &want_packed[(size_t)(slack + count) * packed_width];
          memset(to, 0, packed_width * 2);
          memcpy(to, &hidden[(size_t)r * stride], width * 2);
          top = fmaxf(top, dloss[r]);
          ++count;
        } else if (grad) {
          memset(&want_dhidden[(size_t)r * stride], 0, width * 2);
        } else {
          want_loss[r] = 0.0f;
        }
      }
      if (meta.count != count) fail("count");
      same(index, want_index, "index");
      same(packed, want_packed, "packed rows");
      same(loss, want_loss, "loss");
      same(lse, want_loss, "lse");
      same(dhidden, want_dhidden, "dhidden");
      if (grad && top > 0.0f &&
          !(fabsf(top * meta.scale - 16384.0f) <= 0.01f && fabsf(meta.scale * meta.unscale - 1.0f) <= 1e-6f))
        fail("scale");
    }
  }
  printf("ok\n");
  return 0;
}
