// A warp on the host: 32 lanes as fibers that run in turn from one warp
// intrinsic to the next, where each leaves its operands for the others. Enough
// of CUDA's names for headers that use no more than these.
#pragma once

#include <stdint.h>
#include <ucontext.h>

#include <algorithm>
#include <functional>
#include <memory>
#include <vector>

#define __device__
#define __forceinline__ inline

using std::max;
using std::min;

namespace warp_host {

constexpr int kLanes = 32;
struct State {
  ucontext_t back, lane[kLanes];
  bool done[kLanes];
  uint64_t operand[2][kLanes];  // by the parity of the intrinsic: a lane may be one ahead of the last reader
  int step[kLanes], at;
  const std::function<void(int)>* body;
};
inline State* g_warp;

inline void entry() {
  State& w = *g_warp;
  const int lane = w.at;
  (*w.body)(lane);
  w.done[lane] = true;
  swapcontext(&w.lane[lane], &w.back);
}

// Runs body(lane) as one warp.
inline void run(const std::function<void(int)>& body) {
  auto w = std::make_unique<State>();
  static std::vector<std::vector<char>> stacks(kLanes, std::vector<char>(64 << 10));
  g_warp = w.get();
  w->body = &body;
  for (int l = 0; l < kLanes; ++l) {
    w->done[l] = false;
    w->step[l] = 0;
    getcontext(&w->lane[l]);
    w->lane[l].uc_stack.ss_sp = stacks[l].data();
    w->lane[l].uc_stack.ss_size = stacks[l].size();
    w->lane[l].uc_link = nullptr;
    makecontext(&w->lane[l], entry, 0);
  }
  for (bool some = true; some;) {
    some = false;
    for (int l = 0; l < kLanes; ++l)
      if (!w->done[l]) {
        w->at = l;
        swapcontext(&w->back, &w->lane[l]);
        some = true;
      }
  }
  g_warp = nullptr;
}

// Leaves this lane's operand and comes back when every lane has left its own.
inline const uint64_t* exchange(uint64_t mine) {
  State& w = *g_warp;
  const int lane = w.at, half = w.step[lane]++ & 1;
  w.operand[half][lane] = mine;
  swapcontext(&w.lane[lane], &w.back);
  return w.operand[half];
}

struct ThreadIdx {
  struct X {
    operator int() const { return g_warp->at; }
  } x;
};

}  // namespace warp_host

inline warp_host::ThreadIdx threadIdx;

inline int __shfl_sync(uint32_t, int v, int from) { return int(warp_host::exchange(uint32_t(v))[from & 31]); }
inline int __shfl_up_sync(uint32_t, int v, int by) {
  const int lane = threadIdx.x;
  return int(warp_host::exchange(uint32_t(v))[lane >= by ? lane - by : lane]);
}
inline uint32_t __ballot_sync(uint32_t, bool in) {
  const uint64_t* all = warp_host::exchange(in);
  uint32_t r = 0;
  for (int l = 0; l < 32; ++l) r |= uint32_t(all[l]) << l;
  return r;
}
inline int __reduce_add_sync(uint32_t, int v) {
  const uint64_t* all = warp_host::exchange(uint32_t(v));
  int r = 0;
  for (int l = 0; l < 32; ++l) r += int(all[l]);
  return r;
}
inline int __reduce_max_sync(uint32_t, int v) {
  const uint64_t* all = warp_host::exchange(uint32_t(v));
  int r = int(all[0]);
  for (int l = 1; l < 32; ++l) r = max(r, int(all[l]));
  return r;
}
inline int __popc(uint32_t v) { return __builtin_popcount(v); }
inline int __ffs(uint32_t v) { return __builtin_ffs(int(v)); }
template <typename T>
inline T __ldg(const T* p) {
  return *p;
}
