// CPU counterparts of csrc/block_ops.hpp for the lane emulator (TEST INFRASTRUCTURE ONLY).
#ifndef TCU_BLOCK_OPS_HPP
#define TCU_BLOCK_OPS_HPP

#include <math.h>

#include "wave_ops_emu.hpp"

namespace tcu {

inline float hw_exp2(float x) { return exp2f(x); }
inline float hw_rcp(float x) { return 1.0f / x; }
inline float hw_rsqrt(float x) { return 1.0f / sqrtf(x); }
inline float read_lane_of(float x, int l) {
  auto &w = my_wave();
  w.slot[lane_id()][0] = __float_as_uint(x);
  emu::wave_sync();
  const unsigned r = w.slot[l & 63][0];
  emu::wave_sync();
  return __uint_as_float(r);
}
inline uint16_t bf16_bits(float v) {
  unsigned u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
inline unsigned pack_bf16x2(float lo, float hi) { return (unsigned)bf16_bits(lo) | ((unsigned)bf16_bits(hi) << 16); }

}  // namespace tcu
#endif  // TCU_BLOCK_OPS_HPP
