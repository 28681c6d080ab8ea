// The kernel that moves kept tokens (kernels_evict.hip, cut out of the file by the test), run by a CPU one wave at a time: each
// wave goes from barrier to barrier before the next one starts, in an order that the caller gives.  What one wave may overwrite
// before another has read it is overwritten then.  Lanes of a wave are fibers that meet where lanes exchange values.
#include <ucontext.h>

#include <climits>
#include <cstdint>
#include <cstring>
#include <memory>
#include <vector>

#include "../../tvm_amd/csrc/exact_division.h"

#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(n)
#define __shared__ static
#define __builtin_amdgcn_update_dpp update_dpp
#define __builtin_amdgcn_readlane readlane

struct uint2 { uint32_t x, y; };
struct Index { unsigned x, y, z; };
static uint2 make_uint2(uint32_t x, uint32_t y) { return {x, y}; }
static Index threadIdx, blockIdx, gridDim;
static int min(int a, int b) { return a < b ? a : b; }
static int max(int a, int b) { return a > b ? a : b; }

constexpr int kLanes = 64, kWaves = 4, kThreads = kLanes * kWaves;
enum What { kReady, kAtWave, kAtBarrier, kDone };
struct Fiber {
  ucontext_t context;
  std::unique_ptr<char[]> stack;
  What what;
};
static Fiber fibers[kThreads];
static ucontext_t scheduler;
static int at_wave[kWaves], at_barrier, exchanges[kWaves];
static uint64_t values[kWaves][2][kLanes];

static void pause(What what) {
  const int me = threadIdx.x;
  fibers[me].what = what;
  swapcontext(&fibers[me].context, &scheduler);
}
// All lanes of the wave bring a value and get everyone's.
static const uint64_t* exchange(uint64_t x) {
  const int me = threadIdx.x, wave = me / kLanes;
  uint64_t* const all = values[wave][exchanges[wave] & 1];
  all[me % kLanes] = x;
  if (++at_wave[wave] < kLanes) {
    pause(kAtWave);
  } else {
    at_wave[wave] = 0;
    ++exchanges[wave];
    for (int i = 0; i < kLanes; ++i) {
      if (fibers[wave * kLanes + i].what == kAtWave) fibers[wave * kLanes + i].what = kReady;
    }
  }
  return all;
}
static void __syncthreads() {
  ++at_barrier;
  pause(kAtBarrier);
}
static uint64_t __ballot(bool x) {
  const uint64_t* all = exchange(x);
  uint64_t bits = 0;
  for (int i = 0; i < kLanes; ++i) bits |= all[i] << i;
  return bits;
}
static int readlane(int x, int lane) { return static_cast<int>(exchange(static_cast<uint32_t>(x))[lane]); }
static int update_dpp(int, int x, int control, int, int, bool) {
  const int lane = threadIdx.x % kLanes;
  const uint64_t* all = exchange(static_cast<uint32_t>(x));
  const int from = control == 0xB1 ? lane ^ 1 : control == 0x4E ? lane ^ 2 : control == 0x141 ? lane ^ 7 : lane ^ 15;
  return static_cast<int>(all[from]);
}
static int __popcll(uint64_t x) { return __builtin_popcountll(x); }

namespace tvmkv {
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppRowHalfMirror = 0x141, kDppRowMirror = 0x140;
typedef int int4_any_t __attribute__((ext_vector_type(4), aligned(4)));
union Vec16 { uint32_t w[4]; };
static Vec16 ld16_nt(const void* p) {
  Vec16 v;
  memcpy(&v, p, 16);
  return v;
}
template <int N>
static void wait_vmcnt() {}
#include "move_kept_kernel.inc"
}  // namespace tvmkv

static tvmkv::MoveParams params;
static int which;
static void body() {
  if (which == 0) tvmkv::move_kept_kernel<tvmkv::kMoveInOrder>(params);
  if (which == 1) tvmkv::move_kept_kernel<tvmkv::kMoveFirst>(params);
  if (which == 2) tvmkv::move_kept_kernel<tvmkv::kMoveSecond>(params);
  pause(kDone);
}

// order: the waves, the first to run first.  0, or 1 where some threads wait at a barrier that others never reach.
static int run_workgroup(const int32_t* order) {
  at_barrier = 0;
  for (int w = 0; w < kWaves; ++w) at_wave[w] = 0;
  for (Fiber& f : fibers) {
    if (!f.stack) f.stack.reset(new char[1 << 16]);
    getcontext(&f.context);
    f.context.uc_stack.ss_sp = f.stack.get();
    f.context.uc_stack.ss_size = 1 << 16;
    f.context.uc_link = nullptr;
    f.what = kReady;
    makecontext(&f.context, body, 0);
  }
  for (;;) {
    for (int n = 0; n < kWaves; ++n) {
      for (bool ran = true; ran;) {
        ran = false;
        for (int i = 0; i < kLanes; ++i) {
          const int thread = order[n] * kLanes + i;
          if (fibers[thread].what != kReady) continue;
          ran = true;
          threadIdx = {static_cast<unsigned>(thread), 0, 0};
          swapcontext(&scheduler, &fibers[thread].context);
        }
      }
    }
    int done = 0;
    for (const Fiber& f : fibers) done += f.what == kDone;
    if (done == kThreads) return 0;
    if (done != 0 || at_barrier != kThreads) return 1;
    at_barrier = 0;
    for (Fiber& f : fibers) f.what = kReady;
  }
}

extern "C" int move_kept(int launch, void* pages, float* sums, const int32_t* page_indptr, const int32_t* page_values,
                         const int32_t* weight_page_values, const int32_t* kept, int batch, int h_kv, int max_keep, int page_shift, int pieces,
                         int slices, int parts, const int32_t* order) {
  params.pages = static_cast<uint8_t*>(pages);
  params.key_weights = sums;
  params.page_indptr = page_indptr;
  params.page_values = page_values;
  params.weight_page_values = weight_page_values;
  params.kept = kept;
  params.h_kv = h_kv;
  params.max_keep = max_keep;
  params.page_shift = page_shift;
  params.pieces = pieces;
  params.slices = slices;
  params.by_row = tvmkv::ExactDivision::by(pieces);
  params.by_slice = tvmkv::ExactDivision::by(pieces / slices);
  which = launch;
  gridDim = {static_cast<unsigned>(parts), static_cast<unsigned>(h_kv), static_cast<unsigned>(batch)};
  for (int b = 0; b < batch; ++b) {
    for (int h = 0; h < h_kv; ++h) {
      for (int part = 0; part < parts; ++part) {
        blockIdx = {static_cast<unsigned>(part), static_cast<unsigned>(h), static_cast<unsigned>(b)};
        if (run_workgroup(order) != 0) return 1;
      }
    }
  }
  return 0;
}
