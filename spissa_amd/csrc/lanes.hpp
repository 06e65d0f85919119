// lanes.hpp -- exchanges between the lanes of a wave, the scalar pieces of RoPE and
// the online softmax, and f32 numbers as two binary16 pieces, shared by the kernels.
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

// Max over a wave.
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  v = fmaxf(v, dpp<0x140>(v));
  return max32(max16(v));
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

typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(2))) _Float16 half2v;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

__device__ __forceinline__ float half_lo(unsigned w) { return (float)__builtin_bit_cast(_Float16, (unsigned short)w); }
__device__ __forceinline__ float half_hi(unsigned w) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
}

// Two pieces of eight numbers: the nearest binary16 number and the nearest one of what
// that leaves, so a number within the pieces' range is off by at most 2^-23 of itself, to
// either side. (Cut pieces would be off by up to 2^-21, and always towards zero.)
// (minus_one: -1 as the compiler does not know it, so that the difference is one
// mixed-precision FMA and not a conversion and a subtraction)
__device__ __forceinline__ void split8(const float (&v)[8], float minus_one, half8 *hi, half8 *lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned w = __builtin_bit_cast(unsigned, (half2v){(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
    asm("" : "+v"(w));  // (one packed conversion: the FMAs would have one each again)
    const half2v h = __builtin_bit_cast(half2v, w);
    float r0 = fmaf((float)h.x, minus_one, v[2 * i]), r1 = fmaf((float)h.y, minus_one, v[2 * i + 1]);
    asm("" : "+v"(r0), "+v"(r1));  // (FMAs that write a half of a register each: chunk attention 1 to 2 % slower)
    const half2v l = {(_Float16)r0, (_Float16)r1};
    (*hi)[2 * i] = h.x;
    (*hi)[2 * i + 1] = h.y;
    (*lo)[2 * i] = l.x;
    (*lo)[2 * i + 1] = l.y;
  }
}
// Power of two that takes `most` to 2^top..2^(top + 1), as float bits.
__device__ __forceinline__ unsigned scale_to(float most, unsigned top) {
  return min(254u + top - (__float_as_uint(most) >> 23), 253u) << 23;
}
__device__ __forceinline__ float inverse_scale(unsigned bits) { return __uint_as_float((254u << 23) - bits); }

// Copies 16 bytes a lane from base + off into LDS at lds_base + 16 * lane, unknown
// to the compiler, which would wait for it before any later LDS read: the kernel's
// barriers wait for the copies that the next step reads.
__device__ __forceinline__ void copy16(const char *base, unsigned off, char *lds_base) {
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)lds_base;
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}

}  // namespace
}  // namespace spissa
