// Element types of the recurrent-block operators: 16-byte chunks of fp16, bf16 or fp32 to and from fp32 values, with
// whole-chunk accesses where rows are aligned and element-by-element ones where they are not; activations.
#pragma once

#include "block_ops.hpp"

namespace tcu {

constexpr int kF16 = 0, kBF16 = 1, kF32 = 2;  // tcu_dtype

template <int DT>
struct Elem;
template <>
struct Elem<kF16> {
  using word_t = uint16_t;
  static constexpr int V = 8;  // elements per 16-byte chunk
  TCU_DEVICE static float load(uint16_t w) { return (float)__builtin_bit_cast(half_t, w); }
  TCU_DEVICE static unsigned pack(float lo, float hi) { return pack_f16x2(lo, hi); }
};
template <>
struct Elem<kBF16> {
  using word_t = uint16_t;
  static constexpr int V = 8;
  TCU_DEVICE static float load(uint16_t w) { return __uint_as_float((unsigned)w << 16); }
  TCU_DEVICE static unsigned pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Elem<kF32> {
  using word_t = uint32_t;
  static constexpr int V = 4;
  TCU_DEVICE static float load(uint32_t w) { return __uint_as_float(w); }
};

// chunk -> V fp32 values
template <int DT>
TCU_DEVICE void unpack_chunk(const uint4_t &c, float (&v)[Elem<DT>::V]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const unsigned w = c[i];
    if constexpr (DT == kF32) {
      v[i] = __uint_as_float(w);
    } else {
      v[2 * i] = Elem<DT>::load((uint16_t)(w & 0xffffu));
      v[2 * i + 1] = Elem<DT>::load((uint16_t)(w >> 16));
    }
  }
}
// values 4 q ... 4 q + 3 of a chunk, and four values packed into their place (operators with many operands work on a chunk four
// values at a time, which keeps their operands' fp32 forms from filling the registers)
template <int DT>
TCU_DEVICE void unpack_four(const uint4_t &c, int q, float (&v)[4]) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const unsigned w = c[i];
      v[i] = __uint_as_float(w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const unsigned w = c[2 * q + i];
      v[2 * i] = Elem<DT>::load((uint16_t)(w & 0xffffu));
      v[2 * i + 1] = Elem<DT>::load((uint16_t)(w >> 16));
    }
  }
}
template <int DT>
TCU_DEVICE void pack_four(uint4_t &c, int q, const float (&v)[4]) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) c[2 * q + i] = Elem<DT>::pack(v[2 * i], v[2 * i + 1]);
  }
}
template <int DT>
TCU_DEVICE uint4_t pack_chunk(const float (&v)[Elem<DT>::V]) {
  uint4_t c;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (DT == kF32)
      c[i] = __float_as_uint(v[i]);
    else
      c[i] = Elem<DT>::pack(v[2 * i], v[2 * i + 1]);
  }
  return c;
}

// The chunk at element `at` of p, of which `count` elements exist (count <= 0: none; the others read as 0).
// WHOLE: count is at most 0 or at least V, and p + at is 16-byte aligned.  Otherwise a whole chunk is still one access
// (the hardware takes 16-byte accesses at any element's address), and a part of one is read element by element.
typedef float any_floats_t __attribute__((ext_vector_type(4), aligned(4)));

template <int DT, bool WHOLE, bool NT = true>
TCU_DEVICE uint4_t load_chunk_of(const void *p, size_t at, int count) {
  constexpr int V = Elem<DT>::V;
  const typename Elem<DT>::word_t *q = static_cast<const typename Elem<DT>::word_t *>(p) + at;
  uint4_t c = {0u, 0u, 0u, 0u};
  if (WHOLE ? count > 0 : count >= V) {
    if constexpr (WHOLE && NT) c = __builtin_nontemporal_load(reinterpret_cast<const uint4_t *>(q));
    if constexpr (WHOLE && !NT) c = *reinterpret_cast<const uint4_t *>(q);
    if constexpr (!WHOLE) c = *reinterpret_cast<const any_chunk_t *>(q);  // neighbouring chunks share lines: cached
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < V; e++) {
      if (e < count) {
        const unsigned w = q[e];
        if constexpr (DT == kF32)
          c[e] = w;
        else
          c[e / 2] |= w << (16 * (e % 2));
      }
    }
  }
  return c;
}
template <int DT, bool WHOLE, bool NT = true>
TCU_DEVICE void store_packed(void *p, size_t at, int count, const uint4_t &c) {
  constexpr int V = Elem<DT>::V;
  typename Elem<DT>::word_t *q = static_cast<typename Elem<DT>::word_t *>(p) + at;
  if (WHOLE ? count > 0 : count >= V) {
    if constexpr (WHOLE && NT) __builtin_nontemporal_store(c, reinterpret_cast<uint4_t *>(q));
    if constexpr (WHOLE && !NT) *reinterpret_cast<uint4_t *>(q) = c;
    if constexpr (!WHOLE) *reinterpret_cast<any_chunk_t *>(q) = c;
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < V; e++) {
      if (e < count) {
        if constexpr (DT == kF32)
          q[e] = c[e];
        else
          q[e] = (uint16_t)(c[e / 2] >> (16 * (e % 2)));
      }
    }
  }
}
template <int DT, bool WHOLE, bool NT = true>
TCU_DEVICE void store_chunk_of(void *p, size_t at, int count, const float (&v)[Elem<DT>::V]) {
  if (count > 0) store_packed<DT, WHOLE, NT>(p, at, count, pack_chunk<DT>(v));
}

// V fp32 values at element `at` of a fp32 vector, the same conventions
template <int V, bool WHOLE>
TCU_DEVICE void load_floats(const float *p, size_t at, int count, float (&v)[V]) {
  if (WHOLE ? count > 0 : count >= V) {
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
      float4_t q;
      if constexpr (WHOLE)
        q = *reinterpret_cast<const float4_t *>(p + at + 4 * i);
      else
        q = *reinterpret_cast<const any_floats_t *>(p + at + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * i + e] = q[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = !WHOLE && e < count ? p[at + e] : 0.0f;
  }
}
template <int V, bool WHOLE>
TCU_DEVICE void store_floats(float *p, size_t at, int count, const float (&v)[V]) {
  if (WHOLE ? count > 0 : count >= V) {
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
      const float4_t q = float4_t{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
      if constexpr (WHOLE)
        *reinterpret_cast<float4_t *>(p + at + 4 * i) = q;
      else
        *reinterpret_cast<any_floats_t *>(p + at + 4 * i) = q;
    }
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < V; e++)
      if (e < count) p[at + e] = v[e];
  }
}

// e^x.  EXACT carries the rounding error of x * log2(e) along, a relative error of |x| 2^-24 otherwise.  It is taken where the matrices are
// fp32.  With 16-bit ones, results of 16 bits do not show that error; their fp32 results (states behind a sequence, states of the
// one-token form, gradients of vectors) do carry it: at most |x| / 2 times what the exponential itself may be off, on gates whose own
// rounding to 16 bits moves e^x by up to |x| 2^-8 (bf16) or |x| 2^-11.  The correction would be 6 instructions more on some 26 an element in the scan.
template <bool EXACT>
TCU_DEVICE float exp_of(float x) {
  constexpr float kLog2E = 1.44269504088896340736f, kLog2ELow = 1.92596299112661746887e-8f, kLn2 = 0.69314718055994530942f;
  const float hi = x * kLog2E;
  if constexpr (EXACT) {
    float lo = __builtin_fmaf(x, kLog2E, -hi);
    lo = __builtin_fmaf(x, kLog2ELow, lo);
    const float e = hw_exp2(hi);
    // beyond the range of fp32 (and for an infinite x, whose error term is not a number) e is already the answer
    return __builtin_fabsf(hi) < 128.0f ? __builtin_fmaf(e * lo, kLn2, e) : e;
  }
  return hw_exp2(hi);
}
// s = 1 / (1 + e^-x) and 1 - s, the second as e^-x s: 1 - s would lose the digits that matter where s is close to 1.
// e^-x is held below 2^126 so that both stay finite numbers (a NaN stays a NaN: it fails the comparison).
template <bool EXACT>
TCU_DEVICE void sigmoid_pair(float x, float *s, float *one_minus) {
  const float y = x < -87.0f ? -87.0f : x;
  const float e = exp_of<EXACT>(-y);
  *s = hw_rcp(1.0f + e);
  *one_minus = e * *s;
}

// Activations (tcu_activation) and their slopes.
constexpr int kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActSigmoid = 4;
// The gelu is its tanh form, z (1 + tanh u) / 2 = z sigmoid(2 u) with u = sqrt(2/pi) (z + 0.044715 z^3); so every activation but
// relu is z sigmoid(v) or sigmoid(v).  `act` is the same for all lanes: one branch for a whole array of values.
constexpr float kGeluTwoA = 1.59576912160573071176f, kGeluB = 0.044715f;  // 2 sqrt(2/pi)

// 1 / (1 + e^-x) alone: where e^-x overflows the reciprocal is 0, as it should be
template <bool EXACT>
TCU_DEVICE float sigmoid_of(float x) { return hw_rcp(1.0f + exp_of<EXACT>(-x)); }

// z[] = act(z[])
template <bool EXACT, int N>
TCU_DEVICE void activate(int act, float (&z)[N]) {
  if (act == kActNone) return;
  if (act == kActRelu) {
#pragma unroll
    for (int e = 0; e < N; e++) z[e] = z[e] < 0.0f ? 0.0f : z[e];  // a NaN stays one
  } else if (act == kActSigmoid) {
#pragma unroll
    for (int e = 0; e < N; e++) z[e] = sigmoid_of<EXACT>(z[e]);
  } else if (act == kActSilu) {
#pragma unroll
    for (int e = 0; e < N; e++) z[e] *= sigmoid_of<EXACT>(z[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) z[e] *= sigmoid_of<EXACT>(z[e] * __builtin_fmaf(kGeluTwoA * kGeluB * z[e], z[e], kGeluTwoA));
  }
}
// value[] = act(z[]), slope[] = act'(z[])
template <bool EXACT, int N>
TCU_DEVICE void activate_slope(int act, const float (&z)[N], float (&value)[N], float (&slope)[N]) {
  if (act == kActNone || act == kActRelu) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      value[e] = act == kActRelu && z[e] < 0.0f ? 0.0f : z[e];
      slope[e] = act == kActRelu && !(z[e] > 0.0f) ? 0.0f : 1.0f;
    }
  } else if (act == kActSigmoid) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      float s, r;
      sigmoid_pair<EXACT>(z[e], &s, &r);
      value[e] = s;
      slope[e] = s * r;
    }
  } else if (act == kActSilu) {  // z s(z): s + z s (1 - s)
#pragma unroll
    for (int e = 0; e < N; e++) {
      float s, r;
      const float y = z[e] < -87.0f ? -87.0f : z[e];  // below it the value and the slope are 0 but for 1e-36
      sigmoid_pair<EXACT>(y, &s, &r);
      value[e] = y * s;
      slope[e] = __builtin_fmaf(value[e], r, s);
    }
  } else {  // z s(v): s + z s (1 - s) v'
#pragma unroll
    for (int e = 0; e < N; e++) {
      float s, r;
      // beyond +-32 the sigmoid is 0 or 1, and its argument and v' need not grow any more (they could overflow)
      const float low = z[e] < -32.0f ? -32.0f : z[e], c = low > 32.0f ? 32.0f : low, cz = kGeluTwoA * kGeluB * c;
      sigmoid_pair<EXACT>(c * __builtin_fmaf(cz, c, kGeluTwoA), &s, &r);
      value[e] = low * s;
      slope[e] = __builtin_fmaf(value[e] * r, __builtin_fmaf(3.0f * cz, c, kGeluTwoA), s);
    }
  }
}

// sum of x over the wave, in every lane (a fixed order)
TCU_DEVICE float wave_sum(float x) {
  x += dpp<DPP_QUAD_XOR1>(x, x);
  x += dpp<DPP_QUAD_XOR2>(x, x);
  x += dpp<DPP_ROW_HALF_MIRROR>(x, x);
  x += dpp<DPP_ROW_MIRROR>(x, x);
  return add_xor32(add_xor16(x));
}

}  // namespace tcu
