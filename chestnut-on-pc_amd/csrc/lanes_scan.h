// Sums over the lanes of a wave so far, without LDS.
#pragma once

#include <type_traits>

#include "common.h"

namespace ck {

// Sum over lanes 0..l, in lane l (DPP: six steps without LDS).
template <typename N>
__device__ __forceinline__ N lanes_scan(N v) {
  auto shifted = [](N x, auto CTRL, auto ROWS) {
    return __builtin_bit_cast(N, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(CTRL)::value,
                                                             decltype(ROWS)::value, 0xF, false));
  };
  using std::integral_constant;
  v += shifted(v, integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});   // row_shr:1, 2, 4, 8
  v += shifted(v, integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  v += shifted(v, integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  v += shifted(v, integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  v += shifted(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});   // row_bcast:15, 31
  v += shifted(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return v;
}
__device__ __forceinline__ int lane63(int v) { return __builtin_amdgcn_readlane(v, 63); }

}  // namespace ck
