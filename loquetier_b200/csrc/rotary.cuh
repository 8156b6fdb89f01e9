// The rotary embedding's angles at any position.
#pragma once
#include "smlm_common.cuh"

namespace smlm {

// The 64 frequencies in half-turns per position, base^(-2 i / 128) / pi, each as the sum of two floats.  The pair is good to
// 2^-51 of a half-turn per position, 2^-27 at position 2^24; what rot_sincos adds is the rounding of the reduced angle to one
// float, 2^-24 half-turns.  One float alone is off by several thousandths of a turn from position 10^5 on - more than the
// rounding of a 16-bit result.
struct alignas(16) RotTable {
  float hi[64], lo[64];
};

// A place of the table that a launch carries among its arguments (__grid_constant__), for ordinary loads: lanes that index the
// constant bank at places of their own are served one after another, some 30 cycles each.
__device__ __forceinline__ const float* rot_at(const float* p) {
  asm volatile("" : "+l"(p));
  return p;
}

// cos and sin of pi * pos * (hi + lo) for positions below 2^24 in absolute value; measured up to there, against 64 bits and more:
// off by 2^-20.4 at most (the reduced angle's roundings to a float, and the fast sine)
__device__ __forceinline__ void rot_sincos(float pos, float hi, float lo, float* s, float* c) {
  const float a = __fmul_rn(pos, hi);
  const float e = __fmaf_rn(pos, lo, __fmaf_rn(pos, hi, -a));   // what a lacks
  const float r = a - 2.0f * rintf(0.5f * a) + e;               // the difference of the first two is exact
  *s = __sinf(3.14159265358979f * r);
  *c = __cosf(3.14159265358979f * r);
}


// the table into shared memory, [hi | lo]; every thread of the CTA takes part, a barrier follows at the caller
__device__ __forceinline__ void load_rot_table(const RotTable& rot, float* freq) {
  const float *hi = rot_at(rot.hi), *lo = rot_at(rot.lo);
  for (int i = threadIdx.x; i < 64; i += blockDim.x) {
    freq[i] = hi[i];
    freq[64 + i] = lo[i];
  }
}

}  // namespace smlm
