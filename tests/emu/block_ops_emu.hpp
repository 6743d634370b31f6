// CPU counterparts of csrc/block_ops.hpp for the lane emulator (TEST INFRASTRUCTURE ONLY).
#ifndef TCU_BLOCK_OPS_HPP
#define TCU_BLOCK_OPS_HPP

#include <math.h>

#include "wave_ops_emu.hpp"

namespace tcu {

inline float hw_exp2(float x) { return exp2f(x); }
inline float hw_rcp(float x) { return 1.0f / x; }
inline float hw_rsqrt(float x) { return 1.0f / sqrtf(x); }
template <int D>
inline void swap_halves(unsigned &lo, unsigned &hi) {
  if (D == 16) permlane16_swap(lo, hi);
  else permlane32_swap(lo, hi);
}
typedef unsigned any_chunk_t __attribute__((ext_vector_type(4), aligned(2)));
template <bool WHOLE>
inline uint4_t load_at(const char *base, unsigned offset) {
  if (WHOLE) return *reinterpret_cast<const uint4_t *>(base + offset);
  return *reinterpret_cast<const any_chunk_t *>(base + offset);
}
template <bool WHOLE>
inline void store_at(char *base, unsigned offset, uint4_t v) {
  if (WHOLE) *reinterpret_cast<uint4_t *>(base + offset) = v;
  else *reinterpret_cast<any_chunk_t *>(base + offset) = v;
}
inline float4_t opaque_zero() { return float4_t{0.0f, 0.0f, 0.0f, 0.0f}; }
inline void keep_packed(uint4_t &) {}
inline uint16_t bf16_bits(float v) {
  unsigned u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
inline unsigned pack_bf16x2(float lo, float hi) { return (unsigned)bf16_bits(lo) | ((unsigned)bf16_bits(hi) << 16); }

inline uint2_t read_column_of_four(const half_t *q) {
  auto &w = my_wave();
  const int lane = lane_id();
  memcpy(&w.slot[lane][0], q, 8);
  emu::wave_sync();
  uint16_t column[4];
  for (int r = 0; r < 4; r++) memcpy(&column[r], reinterpret_cast<const char *>(&w.slot[(lane & 48) + 4 * r + (lane & 15) / 4][0]) + 2 * (lane & 3), 2);
  emu::wave_sync();
  uint2_t got;
  memcpy(&got, column, 8);
  return got;
}
template <bool BF16>
inline float4_t mfma_16x16x32_chunks(uint4_t a, uint4_t b, float4_t c) {
  auto &w = my_wave();
  const int lane = lane_id();
  memcpy(&w.slot[lane][0], &a, 16);
  memcpy(&w.slot[lane][4], &b, 16);
  emu::wave_sync();
  auto value = [](const uint32_t *words, int e) {
    const uint16_t h = (uint16_t)(words[e / 2] >> (16 * (e % 2)));
    if (BF16) return __uint_as_float((unsigned)h << 16);
    half_t v;
    memcpy(&v, &h, 2);
    return (float)v;
  };
  float4_t d = c;
  const int n = lane & 15;
  for (int i = 0; i < 4; i++) {
    const int m = 4 * (lane >> 4) + i;
    float acc = 0.0f;
    for (int kb = 0; kb < 4; kb++)
      for (int e = 0; e < 8; e++) acc += value(&w.slot[16 * kb + m][0], e) * value(&w.slot[16 * kb + n][4], e);
    d[i] += acc;
  }
  emu::wave_sync();
  return d;
}

}  // namespace tcu
#endif  // TCU_BLOCK_OPS_HPP
