// Device helpers of the row operators (qknorm.hip, router.hip, logprob.hip): reductions over
// aligned groups of lanes and 16-byte accesses at any element's address.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(4))) unsigned int muon_u4;

template <int CTRL>
MUON_DEVICE uint32_t dpp_move(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}

// op over aligned groups of G lanes, the result in every lane, in a fixed order. Up to 16 lanes
// by DPP, which no LDS port serves: quad permutes, then the mirrors of 8 and of 16 lanes, whose
// halves by then hold equal values. All lanes of a group have to be active.
template <int G, typename T, typename Op>
MUON_DEVICE T group_reduce(T v, Op op) {
  auto moved = [](T x, auto mv) {
    if constexpr (sizeof(T) == 8) {
      const uint64_t b = __builtin_bit_cast(uint64_t, x);
      return __builtin_bit_cast(T, (uint64_t)mv((uint32_t)b) | ((uint64_t)mv((uint32_t)(b >> 32)) << 32));
    } else {
      return __builtin_bit_cast(T, mv(__builtin_bit_cast(uint32_t, x)));
    }
  };
  if constexpr (G >= 2) v = op(v, moved(v, [](uint32_t x) { return dpp_move<0xB1>(x); }));   // xor 1
  if constexpr (G >= 4) v = op(v, moved(v, [](uint32_t x) { return dpp_move<0x4E>(x); }));   // xor 2
  if constexpr (G >= 8) v = op(v, moved(v, [](uint32_t x) { return dpp_move<0x141>(x); }));  // half mirror
  if constexpr (G >= 16) v = op(v, moved(v, [](uint32_t x) { return dpp_move<0x140>(x); })); // mirror
  if constexpr (G >= 32) v = op(v, moved(v, [](uint32_t x) { return (uint32_t)__shfl_xor((int)x, 16, 64); }));
  if constexpr (G >= 64) v = op(v, moved(v, [](uint32_t x) { return (uint32_t)__shfl_xor((int)x, 32, 64); }));
  return v;
}
template <int G>
MUON_DEVICE float group_sum(float v) {
  return group_reduce<G>(v, [](float a, float b) { return a + b; });
}
template <int G>
MUON_DEVICE float group_max(float v) {
  return group_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}

// Values of one 16-byte access: 8 of a two-byte type, 4 of fp32.
template <int DT>
struct Vec16 {
  static constexpr int N = DT == MUON_DT_F32 ? 4 : 8;
  static MUON_DEVICE void unpack(muon_u4 w, float (&v)[N]) {
    if constexpr (DT == MUON_DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == MUON_DT_BF16) {
          v[2 * e] = __uint_as_float(w[e] << 16);
          v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        } else {
          v[2 * e] = f16_to_f32((uint16_t)(w[e] & 0xffffu));
          v[2 * e + 1] = f16_to_f32((uint16_t)(w[e] >> 16));
        }
      }
    }
  }
  static MUON_DEVICE muon_u4 pack(const float (&v)[N]) {
    muon_u4 w;
    if constexpr (DT == MUON_DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(v[e]);
    } else if constexpr (DT == MUON_DT_BF16) {
      // v_cvt_pk_bf16_f32: to nearest even, as f32_to_bf16 (a NaN stays a NaN)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(muon_f2x{v[2 * e], v[2 * e + 1]}, muon_bf2x));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = (uint32_t)f32_to_f16(v[2 * e]) | ((uint32_t)f32_to_f16(v[2 * e + 1]) << 16);
    }
    return w;
  }
};

// 16 bytes at any element's address: the hardware takes them at any byte, so rows of odd
// length need no peeling of their first values.
MUON_DEVICE muon_u4 load_u4(const void* p) {
  muon_u4 w;
  __builtin_memcpy(&w, p, 16);
  return w;
}
MUON_DEVICE void store_u4(void* p, muon_u4 w) { __builtin_memcpy(p, &w, 16); }
// The same past the caches: for results larger than the 256 MB cache, which no store should
// fill with lines that are gone before they are read.
MUON_DEVICE void store_u4_nt(void* p, muon_u4 w) {
  typedef muon_u4 __attribute__((aligned(2))) any_u4;
  __builtin_nontemporal_store(w, (any_u4*)p);
}

template <int DT>
MUON_DEVICE const char* elem_at(const void* p, int64_t i) {
  return (const char*)p + i * (DT == MUON_DT_F32 ? 4 : 2);
}
