// The angles of rotary positions, shared by the kernels that turn heads.
#pragma once

#include "common.h"
#include "elem16.h"

namespace ck {

// A pair's angle is its axis' position times its inverse frequency.
struct RopeAngles {
  const int* pos;          // [T], or one row of T for each of n_axes axes
  const double* inv_freq;  // [half]
  const int* axes;         // [half]: every pair's axis (held to 0 .. n_axes - 1), or null
  int n_axes, T, half;
  float scale, sign;
};

// (scale cos, sign scale sin) of the pairs of tokens t0 .. t0 + nt to LDS, by NT threads.  A
// position of 10^6 makes an angle of 10^6 rad, of which 32 bits hold no more than 0.06 rad: it
// is a product of 64 bits, taken modulo one turn before it is rounded.
template <int NT>
__device__ __forceinline__ void rope_angles(const RopeAngles& p, int t0, int nt, float2_t* cs, int tid) {
  for (int i = tid; i < nt * p.half; i += NT) {
    const int t = i / p.half, pair = i - t * p.half;
    const int* row = p.pos;
    if (p.axes) row += (long)min(max(p.axes[pair], 0), p.n_axes - 1) * p.T;
    double turns = (double)row[t0 + t] * p.inv_freq[pair] * 0.15915494309189533577;
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = float2_t{p.scale * c, p.sign * p.scale * s};
  }
}

}  // namespace ck
