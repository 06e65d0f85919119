// lanes.hpp -- exchanges between the lanes of a wave, and the scalar pieces of
// RoPE and the online softmax, shared by the attention kernels.
#pragma once

#include <hip/hip_runtime.h>

namespace spissa {
namespace {

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false);
}

// Source operand of a DPP add (all source lanes are valid for these controls,
// so `old` is never read; 0 lets the compiler fold it into v_add_f32_dpp).
template <int CTRL>
__device__ __forceinline__ float dpp0(float v) {
  return __builtin_amdgcn_update_dpp(0.0f, v, CTRL, 0xf, 0xf, false);
}

// Sum / max of v with the value of lane ^ 16 or lane ^ 32 (one permlane swap).
__device__ __forceinline__ float sum16(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum32(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max16(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max32(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// All-reduce (sum) over aligned groups of LPR lanes.
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
  static_assert(LPR >= 2 && LPR <= 64 && (LPR & (LPR - 1)) == 0, "LPR");
  v += dpp0<0xB1>(v);                           // lane ^ 1  (quad_perm [1,0,3,2])
  if constexpr (LPR >= 4) v += dpp0<0x4E>(v);   // lane ^ 2  (quad_perm [2,3,0,1])
  if constexpr (LPR >= 8) v += dpp0<0x141>(v);  // quad <-> quad (row_half_mirror)
  if constexpr (LPR >= 16) v += dpp0<0x140>(v); // 8 <-> 8 (row_mirror)
  if constexpr (LPR >= 32) v = sum16(v);        // row <-> row
  if constexpr (LPR >= 64) v = sum32(v);        // half <-> half
  return v;
}

// Max over the row groups of a wave (lanes l, l ^ LPR, l ^ 2 LPR, ...), for a
// value that is uniform within each group of LPR lanes.
template <int LPR>
__device__ __forceinline__ float groups_max(float v) {
  if constexpr (LPR <= 8) v = fmaxf(v, __builtin_amdgcn_update_dpp(v, v, 0x128, 0xf, 0xf, false));  // row_ror:8
  if constexpr (LPR <= 16) v = max16(v);
  if constexpr (LPR <= 32) v = max32(v);
  return v;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ float safe_max(float m) { return m == NEG_INF ? 0.0f : m; }

// rotary.rs:467-481 on one (first, second) pair, each product rounded
// separately, so the result is bit-identical to the reference rotation.
__device__ __forceinline__ void rotate_pair(float &first, float &second, float c, float s) {
#pragma clang fp contract(off)
  const float a = first * c - second * s;
  const float b = second * c + first * s;
  first = a;
  second = b;
}

}  // namespace
}  // namespace spissa
