// linear_q4.hip -- projections of weights held as 4-bit codes with a scale (and
// a zero point) for each group of input channels:
//   out[m, n] = bias[n] + sum_k x[m, k] scale[n, k / group] (code[n, k] - zero[n, k / group]).
//
// Products run on v_mfma_f32_16x16x32_f16. A weight without its scale,
// code - zero, is a whole number of at most 15 and so exact in binary16; an
// activation is scaled by a power of two that takes the largest of its row (or
// of 256 channels of it) to 2^13..2^14, and split into two binary16 pieces, the
// nearest one and the nearest of what is left: 22 bits of each activation down
// to 2^-28 of the largest, and nothing above 2^-38 of the largest is lost. The
// products of a group are summed in f32 and scaled once, so the arithmetic is
// that of f32 sums, at two matrix instructions for 512 weights.
//
// HBM layout, made once when a weight is created: rows in tiles of 16, K in
// blocks of 128. A tile's block is 1 KB of codes in the order in which a wave's
// lanes take them (lane l: row l % 16, quarter l / 16), 16 bytes a lane: four
// words, word j with the eight codes of k = 32 j + 8 (l / 16) + 0..7, codes 2 i
// and 2 i + 1 at bits 4 i and 16 + 4 i, so that a shift and one and-or make a
// pair of binary16 numbers 1024 + code. The block's scales follow the rows:
// [tile][block][row][group in block], zero points beside them (Q4Param).
#include <algorithm>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(2))) _Float16 half2v;
typedef __attribute__((ext_vector_type(4))) _Float16 half4v;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

// A group's scale and zero point as the kernels read them.
//   0: binary16 scale, zero point 8            (2 bytes)
//   1: binary16 scale, binary16 1024 + zero    (4 bytes)
//   2: bfloat16 scale, binary16 1024 + zero    (4 bytes)
//   3: f32 scale, binary16 1024 + zero twice   (8 bytes)
template <int PT>
struct Q4Param {
  static constexpr int BYTES = PT == 0 ? 2 : PT == 3 ? 8 : 4;
};

// The params of a row's block, GPB of them.
template <int PT, int GPB>
struct BlockParams {
  static constexpr int WORDS = (Q4Param<PT>::BYTES * GPB + 3) / 4;
  unsigned w[WORDS];
  __device__ __forceinline__ void load(const char *p) {
    if constexpr (PT == 0 && GPB == 1) {
      w[0] = *reinterpret_cast<const unsigned short *>(p);
    } else if constexpr (WORDS % 4 == 0) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const u32x4 v = reinterpret_cast<const u32x4 *>(p)[i];
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    } else if constexpr (WORDS == 2) {
      const uint2 v = *reinterpret_cast<const uint2 *>(p);
      w[0] = v.x;
      w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const unsigned *>(p);
    }
  }
  __device__ __forceinline__ float scale(int g) const {
    if constexpr (PT == 0)
      return (float)__builtin_bit_cast(_Float16, (unsigned short)(w[g / 2] >> (16 * (g & 1))));
    else if constexpr (PT == 1)
      return (float)__builtin_bit_cast(_Float16, (unsigned short)w[g]);
    else if constexpr (PT == 2)
      return __uint_as_float(w[g] << 16);
    else
      return __uint_as_float(w[2 * g]);
  }
  // 1024 + zero, twice
  __device__ __forceinline__ half2v zero(int g) const {
    if constexpr (PT == 0)
      return (half2v){(_Float16)1032.0f, (_Float16)1032.0f};
    else if constexpr (PT == 3)
      return __builtin_bit_cast(half2v, w[2 * g + 1]);
    else {
      const _Float16 z = __builtin_bit_cast(_Float16, (unsigned short)(w[g] >> 16));
      return (half2v){z, z};
    }
  }
};

// The eight codes of a word less their zero point.
__device__ __forceinline__ half8 weights8(unsigned w, half2v zero) {
  half8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned u = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
    const half2v p = __builtin_bit_cast(half2v, u) - zero;
    r[2 * i] = p.x;
    r[2 * i + 1] = p.y;
  }
  return r;
}

// Power of two that takes a largest |activation| to 2^13..2^14 (as float bits),
// and its inverse.
__device__ __forceinline__ unsigned scale_bits(float most) {
  return min(267u - (__float_as_uint(most) >> 23), 253u) << 23;
}
__device__ __forceinline__ float inverse_scale(unsigned bits) { return __uint_as_float((254u << 23) - bits); }
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;
}
// The two pieces of four scaled activations. An infinity or a NaN is a first
// piece by itself, so that products have what the plain sum would.
__device__ __forceinline__ void split4(const float4 x, float scale, half4v *hi, half4v *lo) {
  const float v[4] = {x.x * scale, x.y * scale, x.z * scale, x.w * scale};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const _Float16 h = (_Float16)v[i];
    (*hi)[i] = h;
    (*lo)[i] = (_Float16)(fabsf(v[i]) <= 65504.0f ? v[i] - (float)h : 0.0f);
  }
}

// x[k..k+3] of a row, zeros from K on. vec: rows are 16-byte aligned.
__device__ __forceinline__ float4 load4(const float *row, int k, int K, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec) {
    if (k < K) v = *reinterpret_cast<const float4 *>(row + k);
  } else {
    if (k < K) v.x = row[k];
    if (k + 1 < K) v.y = row[k + 1];
    if (k + 2 < K) v.z = row[k + 2];
    if (k + 3 < K) v.w = row[k + 3];
  }
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  v = fmaxf(v, dpp<0x140>(v));
  return max32(max16(v));
}

__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace

// Codes, scales and zero points as a checkpoint has them into the layout above.
// One thread per word of codes; the threads of word 0 of a block also make the
// block's params. err: set where a zero point is above 15.
__global__ __launch_bounds__(256) void q4_pack_kernel(const Q4PackArgs a) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long total = (long)a.tiles * a.blocks * 256;
  if (i >= total) return;
  const int j = (int)(i & 3), lane = (int)((i >> 2) & 63);
  const long tb = i >> 8;
  const int block = (int)(tb % a.blocks);
  const long tile = tb / a.blocks;
  const int row = lane & 15, quarter = lane >> 4;
  const long n = tile * 16 + row;
  const int k0 = block * 128 + 32 * j + 8 * quarter;
  const long groups = (a.K + a.group - 1) / a.group;
  const long pitch = ((long)a.K + 1) / 2;
  unsigned word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = k0 + e;
    unsigned c = 8;  // past the matrix: the zero point, a weight of 0
    if (n < a.N && k < a.K) {
      c = (a.codes[n * pitch + k / 2] >> (4 * (k & 1))) & 15u;
    } else if (n < a.N && a.zeros) {
      c = a.zeros[n * groups + min((long)k / a.group, groups - 1)] & 15u;
    }
    word |= c << (4 * (e >> 1) + 16 * (e & 1));
  }
  a.out_codes[i] = word;
  if (quarter == 0 && 32 * j % a.pack_group == 0) {
    const int gpb = 128 / a.pack_group, g = 32 * j / a.pack_group;
    const int k = block * 128 + g * a.pack_group;
    float s = 0.0f;
    unsigned z = 8, sbits = 0;
    if (n < a.N && k < a.K) {  // (groups past K: a scale of 0)
      const long src = n * groups + k / a.group;
      if (a.zeros) z = a.zeros[src];
      if (z > 15) {
        atomicOr(a.err, 1);
        z = 8;
      }
      if (a.scale_dtype == SPISSA_DTYPE_F32) s = reinterpret_cast<const float *>(a.scales)[src];
      else sbits = reinterpret_cast<const unsigned short *>(a.scales)[src];
    }
    const unsigned zb = __builtin_bit_cast(unsigned short, (_Float16)(1024.0f + (float)z));
    const long at = (tb * 16 + row) * gpb + g;
    if (a.param_type == 0) {
      reinterpret_cast<unsigned short *>(a.out_params)[at] = (unsigned short)sbits;
    } else if (a.param_type == 3) {
      reinterpret_cast<uint2 *>(a.out_params)[at] = make_uint2(__float_as_uint(s), zb << 16 | zb);
    } else {
      reinterpret_cast<unsigned *>(a.out_params)[at] = zb << 16 | sbits;
    }
  }
}

// Up to MP (1 or 4) tokens. A wave takes NT row tiles over a range of K blocks;
// the waves of a workgroup are wk ranges x wn runs of tiles. Per 256 channels a
// wave splits its tokens' activations into LDS of its own, in the order in
// which the lanes read them as the matrix instruction's A operand: the 16 rows
// of A repeat the MP tokens, so every lane's accumulators are the same tokens'.
// Bound: HBM for large weights (the codes), latency for small ones.
template <int PT, int GPB, int MP, int NT>
__global__ __launch_bounds__(512) void q4_gemv_kernel(const Q4LinearArgs a) {
  constexpr int KC = 2, SPG = 4 / GPB;  // blocks of a round; 32-deep steps of a group
  __shared__ __attribute__((aligned(16))) half8 xs[8][KC * 4 * 2 * 4 * MP];  // [wave][step][piece][quarter][token]
  __shared__ float red[8][NT * 16][MP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % a.wk, wn = wave / a.wk;
  const int row = lane & 15, quarter = lane >> 4;
  const int runs = (int)(blockDim.x >> 6) / a.wk;
  const long tile0 = ((long)blockIdx.x * runs + wn) * NT;
  const int b0 = wk * a.blocks_per_wave, b1 = min(a.blocks, b0 + a.blocks_per_wave);
  const char *codes[NT], *params[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long tile = min(tile0 + t, (long)a.tiles - 1);  // (tiles past the last are read and not stored)
    codes[t] = reinterpret_cast<const char *>(a.codes) + tile * a.blocks * 1024 + lane * 16;
    params[t] = reinterpret_cast<const char *>(a.params) + (tile * a.blocks * 16 + row) * (GPB * Q4Param<PT>::BYTES);
  }
  constexpr int PB = 16 * GPB * Q4Param<PT>::BYTES;  // bytes of a tile block's params

  float acc[NT][MP];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MP; ++m) acc[t][m] = 0.0f;

  for (int b = b0; b < b1; b += KC) {
    u32x4 w[KC][NT];
    BlockParams<PT, GPB> p[KC][NT];
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const long bb = min(b + c, b1 - 1);  // (a block past the range is not used)
        w[c][t] = *reinterpret_cast<const u32x4 *>(codes[t] + bb * 1024);
        p[c][t].load(params[t] + bb * PB);
      }
    // Four channels a lane and token: step lane / 8 (of 32 channels), quarter
    // (lane / 2) % 4, half lane % 2 of its eight.
    float inv[MP];
#pragma unroll
    for (int m = 0; m < MP; ++m) {
      const int tok = min(m, a.M - 1);
      const float4 v = load4(a.x + (long)tok * a.K, b * 128 + 4 * lane, min(a.K, b1 * 128), a.vec);
      const float most = wave_max(fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))));
      const unsigned sb = scale_bits(most);
      inv[m] = inverse_scale(sb);
      half4v hi, lo;
      split4(v, __uint_as_float(sb), &hi, &lo);
      half4v *dst = reinterpret_cast<half4v *>(&xs[wave][((lane >> 3) * 2 * 4 + ((lane >> 1) & 3)) * MP + m]) + (lane & 1);
      dst[0] = hi;
      dst[4 * MP * 2] = lo;
    }
    wave_lds_order();
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      if (b + c >= b1) break;
      f32x4 sum[NT];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const half8 hi = xs[wave][((c * 4 + j) * 2 * 4 + quarter) * MP + row % MP];
        const half8 lo = xs[wave][(((c * 4 + j) * 2 + 1) * 4 + quarter) * MP + row % MP];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const half8 wf = weights8(w[c][t][j], p[c][t].zero(j / SPG));
          if (j % SPG == 0) sum[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
          sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, wf, sum[t], 0, 0, 0);
          sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, wf, sum[t], 0, 0, 0);
          if (j % SPG == SPG - 1) {
            const float s = p[c][t].scale(j / SPG);
#pragma unroll
            for (int m = 0; m < MP; ++m) acc[t][m] = fmaf(sum[t][m], s * inv[m], acc[t][m]);
          }
        }
      }
    }
    wave_lds_order();
  }
  // The ranges' sums, in range order (the four quarters hold the same).
  if (quarter == 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MP; ++m) red[wave][t * 16 + row][m] = acc[t][m];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < runs * NT * 16; i += blockDim.x) {
    const int r = i / (NT * 16), o = i - r * (NT * 16);
    const long n = ((long)blockIdx.x * runs + r) * NT * 16 + o;
    if (n >= a.N) continue;
    const float bias = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int m = 0; m < MP; ++m) {
      if (m >= a.M) break;
      float v = 0.0f;
      for (int q = 0; q < a.wk; ++q) v += red[r * a.wk + q][o][m];
      a.out[(long)m * a.N + n] = v + bias;
    }
  }
}

// The pieces of every token's activations in the order of the A operand,
// [row tile][32-deep step][piece][lane], and the inverse of its scale. One
// workgroup a token (rows past the last are zeros).
__global__ __launch_bounds__(256) void q4_pieces_kernel(const float *x, int M, int K, int steps, bool vec, half8 *pieces,
                                                        float *inv) {
  __shared__ float part[4];
  const int m = blockIdx.x, tid = threadIdx.x;
  const float *row = x + (long)min(m, M - 1) * K;
  float most = 0.0f;
  for (int k = 4 * tid; k < K; k += 1024) {
    const float4 v = load4(row, k, K, vec);
    most = fmaxf(most, fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))));
  }
  most = wave_max(most);
  if ((tid & 63) == 0) part[tid >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const unsigned sb = scale_bits(most);
  if (tid == 0) inv[m] = inverse_scale(sb);
  half8 *dst = pieces + (long)(m >> 4) * steps * 128;
  for (int u = tid; u < steps * 4; u += 256) {  // eight channels: step u / 4, quarter u % 4
    half8 h{}, l{};
    if (m < M) {
      half4v h0, l0, h1, l1;
      split4(load4(row, 8 * u, K, vec), __uint_as_float(sb), &h0, &l0);
      split4(load4(row, 8 * u + 4, K, vec), __uint_as_float(sb), &h1, &l1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = h0[i];
        h[4 + i] = h1[i];
        l[i] = l0[i];
        l[4 + i] = l1[i];
      }
    }
    half8 *at = dst + (long)(u >> 2) * 128 + (u & 3) * 16 + (m & 15);
    at[0] = h;
    at[64] = l;
  }
}

// More tokens: a wave takes MT x NT tiles of 16 x 16 outputs over a range of K
// blocks (the waves of a workgroup: wk ranges x wn runs of row tiles of the
// weight), both operands straight from memory.
template <int PT, int GPB, int MT, int NT>
__global__ __launch_bounds__(256) void q4_tile_kernel(const Q4LinearArgs a) {
  constexpr int SPG = 4 / GPB, PB = 16 * GPB * Q4Param<PT>::BYTES;
  extern __shared__ __attribute__((aligned(16))) float red[];  // [wave][MT * NT][4][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % a.wk, wn = wave / a.wk, runs = 4 / a.wk;
  const int row = lane & 15, quarter = lane >> 4;
  const long tile0 = ((long)blockIdx.x * runs + wn) * NT;
  const int mt0 = blockIdx.y * MT;
  const int b0 = wk * a.blocks_per_wave, b1 = min(a.blocks, b0 + a.blocks_per_wave);
  const char *codes[NT], *params[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long tile = min(tile0 + t, (long)a.tiles - 1);
    codes[t] = reinterpret_cast<const char *>(a.codes) + tile * a.blocks * 1024 + lane * 16;
    params[t] = reinterpret_cast<const char *>(a.params) + (tile * a.blocks * 16 + row) * (GPB * Q4Param<PT>::BYTES);
  }
  const half8 *xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xp[i] = reinterpret_cast<const half8 *>(a.pieces) + (long)min(mt0 + i, a.mtiles - 1) * a.blocks * 512 + lane;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int b = b0; b < b1; ++b) {
    u32x4 w[NT];
    BlockParams<PT, GPB> p[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w[t] = *reinterpret_cast<const u32x4 *>(codes[t] + (long)b * 1024);
      p[t].load(params[t] + (long)b * PB);
    }
    f32x4 sum[MT][NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      half8 hi[MT], lo[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        hi[i] = xp[i][(b * 4 + j) * 128];
        lo[i] = xp[i][(b * 4 + j) * 128 + 64];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const half8 wf = weights8(w[t][j], p[t].zero(j / SPG));
        const float s = p[t].scale(j / SPG);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (j % SPG == 0) sum[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
          sum[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[i], wf, sum[i][t], 0, 0, 0);
          sum[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[i], wf, sum[i][t], 0, 0, 0);
          if (j % SPG == SPG - 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(sum[i][t][e], s, acc[i][t][e]);
          }
        }
      }
    }
  }
  if (a.wk > 1) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[((wave * MT * NT + i * NT + t) * 4 + e) * 64 + lane] = acc[i][t][e];
    __syncthreads();
    if (wk != 0) return;
    for (int q = 1; q < a.wk; ++q)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][t][e] += red[(((wave + q) * MT * NT + i * NT + t) * 4 + e) * 64 + lane];
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long n = (tile0 + t) * 16 + row;
    if (n >= a.N) continue;
    const float bias = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long m = (long)(mt0 + i) * 16 + 4 * quarter + e;
        if (m < a.M) a.out[m * a.N + n] = fmaf(acc[i][t][e], a.inv[m], bias);
      }
  }
}

namespace {

template <int PT, int GPB>
hipError_t run(hipStream_t st, Q4LinearArgs a) {
  if (a.M <= 4) {
    // Waves of a workgroup share K while tiles are few.
    const int rounds = (a.blocks + 1) / 2;
    a.wk = 1;
    while (a.wk < 8 && a.wk < rounds && (long)a.tiles * a.wk < 2048) a.wk *= 2;
    a.blocks_per_wave = ((rounds + a.wk - 1) / a.wk) * 2;
    const int waves = std::max(4, a.wk), runs = waves / a.wk;
    const dim3 grid((unsigned)((a.tiles + runs - 1) / runs));
    if (a.M == 1) hipLaunchKernelGGL((q4_gemv_kernel<PT, GPB, 1, 1>), grid, dim3(waves * 64), 0, st, a);
    else hipLaunchKernelGGL((q4_gemv_kernel<PT, GPB, 4, 1>), grid, dim3(waves * 64), 0, st, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(q4_pieces_kernel, dim3((unsigned)(a.mtiles * 16)), dim3(256), 0, st, a.x, a.M, a.K, a.blocks * 4, a.vec,
                     (half8 *)a.pieces, (float *)a.inv);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.M <= 32) {
    a.wk = std::min(4, a.blocks >= 4 ? 4 : a.blocks >= 2 ? 2 : 1);
    a.blocks_per_wave = (a.blocks + a.wk - 1) / a.wk;
    const int runs = 4 / a.wk;
    const dim3 grid((unsigned)((a.tiles + runs - 1) / runs), (unsigned)a.mtiles);
    hipLaunchKernelGGL((q4_tile_kernel<PT, GPB, 1, 1>), grid, dim3(256), 4 * 4 * 64 * 4, st, a);
  } else {
    a.wk = 1;
    a.blocks_per_wave = a.blocks;
    const dim3 grid((unsigned)((a.tiles + 15) / 16), (unsigned)((a.mtiles + 3) / 4));
    hipLaunchKernelGGL((q4_tile_kernel<PT, GPB, 4, 4>), grid, dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

template <int PT>
hipError_t run_g(hipStream_t st, const Q4LinearArgs &a, int group) {
  switch (group) {
    case 32: return run<PT, 4>(st, a);
    case 64: return run<PT, 2>(st, a);
    case 128: return run<PT, 1>(st, a);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

size_t q4_param_bytes(int param_type) { return param_type == 0 ? 2 : param_type == 3 ? 8 : 4; }

hipError_t launch_q4_pack(hipStream_t st, const Q4PackArgs &a) {
  const long total = (long)a.tiles * a.blocks;
  hipLaunchKernelGGL(q4_pack_kernel, dim3((unsigned)total), dim3(256), 0, st, a);
  return hipGetLastError();
}

// Bytes of the activations' pieces and inverse scales that M tokens need (0: none).
size_t q4_linear_workspace(long M, long blocks) {
  if (M <= 4) return 0;
  const size_t mt = (size_t)(M + 15) / 16;
  return mt * blocks * 8192 + mt * 16 * sizeof(float);
}

hipError_t launch_q4_linear(hipStream_t st, const Q4LinearArgs &base, int group, int param_type, void *workspace) {
  Q4LinearArgs a = base;
  a.mtiles = (a.M + 15) / 16;
  a.vec = a.K % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  a.pieces = workspace;
  a.inv = reinterpret_cast<const float *>(static_cast<char *>(workspace) + (size_t)a.mtiles * a.blocks * 8192);
  switch (param_type) {
    case 0: return run_g<0>(st, a, group);
    case 1: return run_g<1>(st, a, group);
    case 2: return run_g<2>(st, a, group);
    case 3: return run_g<3>(st, a, group);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace spissa
