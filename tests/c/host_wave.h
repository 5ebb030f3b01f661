// A wave of 64 lanes on the host, for device headers whose lanes work together
// by ballots, shuffles and lane reads alone: each lane is a context of its own,
// and a lane that reaches a collective waits there until all have.  Stands in for
// csrc/kernels/common.h.
#pragma once

#include <setjmp.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <ucontext.h>

#include <functional>
#include <vector>

#define __device__
#define __forceinline__ inline

namespace bwpp {}

namespace host_wave {

constexpr int kLanes = 64;
constexpr size_t kStack = 64 * 1024;

struct Dim {
  uint32_t x = 0, y = 0, z = 0;
};

inline Dim thread, block;
inline ucontext_t lanes[kLanes];  // a lane's first switch; then by jumps, without system calls
inline jmp_buf scheduler, at[kLanes];
inline bool begun[kLanes];
inline uint64_t values[2][kLanes];  // of the last two collectives
inline uint64_t count[kLanes];      // collectives of a lane
inline bool done[kLanes];
inline const std::function<void()> *body;

// Every lane's value of one collective (valid until the lane's next one).
inline const uint64_t *all(uint64_t v) {
  const int lane = (int)thread.x;
  uint64_t *row = values[count[lane]++ & 1u];
  row[lane] = v;
  if (!_setjmp(at[lane])) _longjmp(scheduler, 1);
  return row;
}

inline void entry() {
  (*body)();
  done[thread.x] = true;
  _longjmp(scheduler, 1);
}

// Runs f in every lane of one wave.  All lanes have to reach the same collectives.
inline void run(uint32_t block_x, const std::function<void()> &f) {
  static std::vector<char> stacks(kLanes * kStack);
  body = &f;
  block.x = block_x;
  for (int i = 0; i < kLanes; ++i) {
    getcontext(&lanes[i]);
    lanes[i].uc_stack.ss_sp = stacks.data() + (size_t)i * kStack;
    lanes[i].uc_stack.ss_size = kStack;
    lanes[i].uc_link = nullptr;
    makecontext(&lanes[i], entry, 0);
    count[i] = 0;
    begun[i] = done[i] = false;
  }
  for (;;) {
    for (volatile int i = 0; i < kLanes; ++i) {
      thread.x = (uint32_t)i;
      if (_setjmp(scheduler)) continue;
      if (begun[i]) _longjmp(at[i], 1);
      begun[i] = true;
      setcontext(&lanes[i]);
    }
    for (int i = 1; i < kLanes; ++i)
      if (done[i] != done[0] || count[i] != count[0]) {
        fprintf(stderr, "lanes %d and 0 part ways in block %u\n", i, block_x);
        exit(2);
      }
    if (done[0]) return;
  }
}

}  // namespace host_wave

#define threadIdx host_wave::thread
#define blockIdx host_wave::block

inline uint64_t __ballot(bool p) {
  const uint64_t *v = host_wave::all(p);
  uint64_t bits = 0;
  for (int i = 0; i < host_wave::kLanes; ++i) bits |= (v[i] & 1u) << i;
  return bits;
}
inline uint64_t __shfl_up(uint64_t v, int d, int) {
  const int lane = (int)threadIdx.x;
  return host_wave::all(v)[lane >= d ? lane - d : lane];
}
inline int __builtin_amdgcn_readlane(int v, int lane) { return (int)host_wave::all((uint32_t)v)[lane]; }
inline int __builtin_amdgcn_readfirstlane(int v) { return (int)host_wave::all((uint32_t)v)[0]; }
inline void __syncthreads() { host_wave::all(0); }
inline int __syncthreads_or(int p) { return __ballot(p != 0) != 0; }

template <class T>
inline T min(T a, T b) {
  return b < a ? b : a;
}
template <class T>
inline T max(T a, T b) {
  return a < b ? b : a;
}
