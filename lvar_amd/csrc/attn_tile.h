// What the kernels of the attention share: the schedule of a tile's softmax, compile-time loops, waits for LDS fills.
#pragma once
#include <type_traits>
#include "common.h"

namespace lvar {

constexpr int READ_AHEAD = 4;    // operand fragments requested from LDS this many MFMAs before their use
constexpr int EXP_IN_QK = 24;    // of the 32 exp2 per lane and tile, how many run next to the QK MFMAs

// First S element of softmax slot g: EA elements spread over the NQK steps of the QK phase, the other
// 32 - EA over the first HB steps of the PV phase; slots before 0 and after the last one are empty.
template <int NQK, int HB, int EA>
struct ExpSlots {
  static constexpr int lo(int g) {
    return g <= 0 ? 0 : g < NQK ? g * EA / NQK : g < NQK + HB ? EA + (g - NQK) * (32 - EA) / (HB ? HB : 1) : 32;
  }
};

// f(integral_constant<int, i>) for i = LO .. HI-1, unrolled at compile time
template <int LO, int HI, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (LO < HI) {
    f(std::integral_constant<int, LO>{});
    static_for<LO + 1, HI>(f);
  }
}
static constexpr float RESCALE_TAU = 8.0f;
static constexpr float NEG_BIG = -1.0e30f;

#if defined(__HIP_DEVICE_COMPILE__)

// Wait until at most N of this wave's global reads and LDS fills are outstanding (they complete in order)
template <int N>
__device__ __forceinline__ void wait_fills() {
  static_assert(N < 64, "six bits of the counter");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

// x, never fused with what is added to it: whether the compiler would depends on the instance, and all have the same bits
__device__ __forceinline__ float rounded(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

#endif

}  // namespace lvar
