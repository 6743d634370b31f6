// What the recurrent-block operators (gated scan, fused norm, fused matrix product) use beyond wave_ops.hpp: element
// types behind a 16-byte chunk, the transcendental instructions, lane exchanges.
//
// A chunk is 16 bytes of one row: 8 elements of 16 bits or 4 of 32.  Everything is computed in fp32; the one rounding to
// 16 bits is the conversion of a result to the type its tensor has (to nearest even).
#ifndef TCU_BLOCK_OPS_HPP
#define TCU_BLOCK_OPS_HPP

#include "wave_ops.hpp"

namespace tcu {

// 2^x, 1/x, 1/sqrt(x): the hardware's instructions, within 1 ulp (results below 2^-126 are 0)
TCU_DEVICE float hw_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
TCU_DEVICE float hw_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
TCU_DEVICE float hw_rsqrt(float x) { return __builtin_amdgcn_rsqf(x); }

// With lo = hi = x: lo becomes x of the lane without bit D in its number, hi x of the lane with it (D = 16 or 32)
template <int D>
TCU_DEVICE void swap_halves(unsigned &lo, unsigned &hi) {
  if constexpr (D == 16) permlane16_swap(lo, hi);
  else permlane32_swap(lo, hi);
}

// 16 bytes at a 32-bit offset from a base that is the same for the whole wave (which then stays in scalar registers).
// WHOLE: 16-byte aligned; otherwise at any element's address.
typedef unsigned any_chunk_t __attribute__((ext_vector_type(4), aligned(2)));
template <bool WHOLE>
TCU_DEVICE uint4_t load_at(const char *base, unsigned offset) {
  if constexpr (WHOLE) return __builtin_nontemporal_load(reinterpret_cast<const uint4_t *>(base + offset));
  return *reinterpret_cast<const any_chunk_t *>(base + offset);
}
template <bool WHOLE>
TCU_DEVICE void store_at(char *base, unsigned offset, uint4_t v) {
  if constexpr (WHOLE) __builtin_nontemporal_store(v, reinterpret_cast<uint4_t *>(base + offset));
  else *reinterpret_cast<any_chunk_t *>(base + offset) = v;
}

// Hides from the compiler that `c` is what it was: what is unpacked from it is then not kept across a loop in twice the registers.
TCU_DEVICE void keep_packed(uint4_t &c) { asm volatile("" : "+v"(c)); }

// four zeros that the compiler does not know to be zeros
TCU_DEVICE float4_t opaque_zero() {
  float4_t z = {0.0f, 0.0f, 0.0f, 0.0f};
  asm volatile("" : "+v"(z));
  return z;
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
TCU_DEVICE unsigned pack_bf16x2(float lo, float hi) {
  bf16x2_t v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(unsigned, v);
}

// D = A B + C on 16x16x32 MFMAs of either 16-bit type, operands as 16-byte chunks (layouts: wave_ops.hpp)
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
template <bool BF16>
TCU_DEVICE float4_t mfma_16x16x32_chunks(uint4_t a, uint4_t b, float4_t c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return mfma_16x16x32(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c);
}

// 16 lanes read a block of 4 rows of 16 elements of 16 bits, lane 4 r + c the elements 4 c ... 4 c + 3 of row r (8 bytes at `q`);
// lane i gets column i of it.
TCU_DEVICE uint2_t read_column_of_four(const half_t *q) {
  typedef short short4_t __attribute__((ext_vector_type(4)));
  using lds_ptr_t = __attribute__((address_space(3))) short4_t *;
  return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(uintptr_t)lds_address_of(q)));
}

}  // namespace tcu
#endif  // TCU_BLOCK_OPS_HPP
