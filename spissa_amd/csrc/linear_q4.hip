// linear_q4.hip -- projections of weights held as 4-bit codes with a scale (and
// a zero point) for each group of input channels:
//   out[m, n] = bias[n] + sum_k x[m, k] scale[n, k / group] (code[n, k] - zero[n, k / group]).
//
// Products run on v_mfma_f32_16x16x32_f16. A weight without its scale,
// code - zero, is a whole number of at most 15 and so exact in binary16; an
// activation is scaled by a power of two that takes the largest of its row (or
// of 512 channels of it) to 2^13..2^14, and split into two binary16 pieces, the
// nearest one and the nearest of what is left: off by at most 2^-23 of each
// activation down to 2^-15 of the largest, and below by at most 2^-38 of the
// largest, where the second piece's last digit is. The products of a group are
// summed in f32 and scaled once, so the arithmetic is that of f32 sums, at two
// matrix instructions for 512 weights.
//
// HBM layout, made once when a weight is created: rows in tiles of 16, K in
// blocks of 128. A tile's block is 1 KB of codes in the order in which a wave's
// lanes take them (lane l: row l % 16, quarter l / 16), 16 bytes a lane: four
// words, word j with the eight codes of k = 32 j + 8 (l / 16) + 0..7, codes 2 i
// and 2 i + 1 at bits 4 i and 16 + 4 i: read as binary16 numbers, those in bits 0..3
// are code 2^-24 and those in bits 4..7 code 2^-20, so that one packed FMA makes a
// pair of weights (code - zero) 2^-9, exactly; the 2^9 is in the tokens' factors. The block's scales follow the rows:
// [tile][block][row][group in block], zero points beside them (Q4Param).
#include <algorithm>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

typedef __attribute__((ext_vector_type(4))) _Float16 half4v;

// A group's scale and zero point as the kernels read them.
//   0: binary16 scale, zero point 8            (2 bytes)
//   1: binary16 scale, binary16 -zero / 512    (4 bytes)
//   2: bfloat16 scale, binary16 -zero / 512    (4 bytes)
//   3: f32 scale, binary16 -zero / 512 twice   (8 bytes)
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
  __device__ __forceinline__ void here() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[i]));
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
  // -zero / 512, twice
  __device__ __forceinline__ half2v zero(int g) const {
    if constexpr (PT == 0)
      return (half2v){(_Float16)-0x1p-6f, (_Float16)-0x1p-6f};
    else if constexpr (PT == 3)
      return __builtin_bit_cast(half2v, w[2 * g + 1]);
    else {
      const _Float16 z = __builtin_bit_cast(_Float16, (unsigned short)(w[g] >> 16));
      return (half2v){z, z};
    }
  }
};

// The factors of codes in bits 0..3 and 4..7, 2^15 and 2^11 twice, as values that the
// compiler does not know (it would take shifts for them).
struct Factors {
  half2v from0, from4;
  __device__ __forceinline__ Factors() {
    unsigned a = 0x78007800u, b = 0x68006800u;
    asm volatile("" : "+v"(a), "+v"(b));
    from0 = __builtin_bit_cast(half2v, a);
    from4 = __builtin_bit_cast(half2v, b);
  }
};
// The eight codes of a word less their zero point, times 2^-9.
__device__ __forceinline__ half8 weights8(unsigned w, half2v zero, const Factors &f) {
  half8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned u = (i & 2 ? w >> 8 : w) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
    const half2v p = __builtin_elementwise_fma(__builtin_bit_cast(half2v, u), i & 1 ? f.from4 : f.from0, zero);
    r[2 * i] = p.x;
    r[2 * i + 1] = p.y;
  }
  return r;
}

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
    const unsigned zb = __builtin_bit_cast(unsigned short, (_Float16)((float)z * (-1.0f / 512.0f)));
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

// The weights and params of a block of NT tiles, as a lane has them.
template <int PT, int GPB, int NT>
struct BlockWeights {
  u32x4 w[NT];
  BlockParams<PT, GPB> p[NT];
  __device__ __forceinline__ void load(const char *const (&codes)[NT], const char *const (&params)[NT], long block) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w[t] = *reinterpret_cast<const u32x4 *>(codes[t] + block * 1024);
      p[t].load(params[t] + block * (16 * GPB * Q4Param<PT>::BYTES));
    }
  }
  __device__ __forceinline__ void here() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      asm volatile("" : "+v"(w[t]));
      p[t].here();
    }
  }
};

// acc += the block's products with the A fragments hi, lo (rows 4 (lane / 16) + 0..3
// of A), the first E rows of the lane's four.
template <int PT, int GPB, int NT, int E, typename FRAGS, typename INV>
__device__ __forceinline__ void block_products(const BlockWeights<PT, GPB, NT> &b, const Factors &factors, FRAGS frags, const INV &inv,
                                               float (&acc)[NT][E]) {
  constexpr int SPG = 4 / GPB;  // 32-deep steps of a group
  f32x4 sum[NT];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    half8 hi, lo;
    frags(j, &hi, &lo);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const half8 wf = weights8(b.w[t][j], b.p[t].zero(j / SPG), factors);
      if (j % SPG == 0) sum[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
      sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, wf, sum[t], 0, 0, 0);
      sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, wf, sum[t], 0, 0, 0);
      if (j % SPG == SPG - 1) {
        const float s = b.p[t].scale(j / SPG);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[t][e] = fmaf(sum[t][e], s * inv[e], acc[t][e]);
      }
    }
  }
}

// A lane's tiles: where their codes and params begin. (Tiles past the last are
// read as the last and not stored.)
template <int PT, int GPB, int NT>
__device__ __forceinline__ void tile_addresses(const Q4LinearArgs &a, long tile0, int lane, const char *(&codes)[NT],
                                               const char *(&params)[NT]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long tile = min(tile0 + t, (long)a.tiles - 1);
    codes[t] = reinterpret_cast<const char *>(a.codes) + tile * a.blocks * 1024 + lane * 16;
    params[t] =
        reinterpret_cast<const char *>(a.params) + (tile * a.blocks * 16 + (lane & 15)) * (GPB * Q4Param<PT>::BYTES);
  }
}

// Up to MP (1 or 4) tokens. A wave takes NT row tiles over a range of K blocks;
// the waves of a workgroup are wk ranges x runs of tiles. Per 512 channels a
// wave splits its tokens' activations into LDS of its own, in the order in
// which the lanes read them as the matrix instruction's A operand: the 16 rows
// of A repeat the MP tokens, so every lane's accumulators are the same tokens'.
// The codes and activations of the next 512 channels are in flight meanwhile.
// Bound: HBM for large weights (the codes), latency for small ones. One token: 262144 x
// 1152 35 us, 4.6 TB/s; 16384 x 4096 10 us; 4096 x 4096 5.2 us; 2048 x 8192 5.9 us; two
// to four tokens, 4096 x 4096 7.5 to 7.7 us.
template <int PT, int GPB, int MP, int NT>
__global__ __launch_bounds__(MP == 1 ? 1024 : 512) void q4_gemv_kernel(const Q4LinearArgs a) {
  constexpr int KC = 4;  // blocks of a round
  constexpr int WAVES = MP == 1 ? 16 : 8;
  __shared__ __attribute__((aligned(16))) half8 xs[WAVES][KC * 4 * 2 * 4 * MP];  // [wave][step][piece][quarter][token]
  __shared__ float red[WAVES][NT * 16][MP];
  const Factors factors;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % a.wk, wn = wave / a.wk;
  const int row = lane & 15, quarter = lane >> 4;
  const int runs = (int)(blockDim.x >> 6) / a.wk;
  const long tile0 = ((long)blockIdx.x * runs + wn) * NT;
  const int b0 = wk * a.blocks_per_wave, b1 = min(a.blocks, b0 + a.blocks_per_wave);
  const char *codes[NT], *params[NT];
  tile_addresses<PT, GPB, NT>(a, tile0, lane, codes, params);

  float acc[NT][MP];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MP; ++m) acc[t][m] = 0.0f;

  BlockWeights<PT, GPB, NT> w[KC];
  float4 xv[MP][2];
  auto load_w = [&](int b) {
#pragma unroll
    for (int c = 0; c < KC; ++c) w[c].load(codes, params, min(b + c, b1 - 1));  // (blocks past the range are not used)
  };
  // Eight channels a lane and token: step lane / 4 (of 32 channels), quarter lane % 4.
  auto load_x = [&](int b) {
#pragma unroll
    for (int m = 0; m < MP; ++m) {
      const float *xr = a.x + (long)min(m, a.M - 1) * a.K;
      const int k = b * 128 + 8 * lane, end = min(a.K, b1 * 128);
      xv[m][0] = load4(xr, k, end, a.vec);
      xv[m][1] = load4(xr, k + 4, end, a.vec);
    }
  };
  if (b0 < b1) {
    load_x(b0);
    load_w(b0);
  }
  for (int b = b0; b < b1; b += KC) {
    float inv[MP];
#pragma unroll
    for (int m = 0; m < MP; ++m) {
      const float4 u = xv[m][0], v = xv[m][1];
      const float most =
          wave_max(fmaxf(fmaxf(fmaxf(finite_abs(u.x), finite_abs(u.y)), fmaxf(finite_abs(u.z), finite_abs(u.w))),
                         fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w)))));
      const unsigned sb = scale_to(most, 13);
      inv[m] = 512.0f * inverse_scale(sb);
      half4v h[2], l[2];
      split4(u, __uint_as_float(sb), &h[0], &l[0]);
      split4(v, __uint_as_float(sb), &h[1], &l[1]);
      half8 *dst = &xs[wave][((lane >> 2) * 2 * 4 + (lane & 3)) * MP + m];
      dst[0] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
      dst[4 * MP] = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const bool more = b + KC < b1;
    if (more) load_x(b + KC);
    wave_lds_order();
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      if (b + c >= b1) break;
      auto frags = [&](int j, half8 *hi, half8 *lo) {
        *hi = xs[wave][((c * 4 + j) * 2 * 4 + quarter) * MP + row % MP];
        *lo = xs[wave][(((c * 4 + j) * 2 + 1) * 4 + quarter) * MP + row % MP];
      };
      block_products<PT, GPB, NT, MP>(w[c], factors, frags, inv, acc);
      if (more) w[c].load(codes, params, min(b + KC + c, b1 - 1));
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
// workgroup of 1024 for T tokens (rows past the last are zeros), T neighbours of a
// row tile a 16 T byte store; the first 8192 / T channels of a row are read once.
template <int T>
__global__ __launch_bounds__(1024) void q4_pieces_kernel(const float *x, int M, int K, int steps, bool vec, half8 *pieces,
                                                         float *inv) {
  __shared__ float part[16][T];
  const int tid = threadIdx.x, r = tid % T, unit = tid / T, m = blockIdx.x * T + r;
  const float *row = x + (long)min(m, M - 1) * K;
  float4 u = load4(row, 8 * unit, K, vec), v = load4(row, 8 * unit + 4, K, vec);
  auto most_of = [](const float4 &a, const float4 &b) {
    return fmaxf(fmaxf(fmaxf(finite_abs(a.x), finite_abs(a.y)), fmaxf(finite_abs(a.z), finite_abs(a.w))),
                 fmaxf(fmaxf(finite_abs(b.x), finite_abs(b.y)), fmaxf(finite_abs(b.z), finite_abs(b.w))));
  };
  float most = most_of(u, v);
  for (int k = 8 * (unit + 1024 / T); k < K; k += 8192 / T)
    most = fmaxf(most, most_of(load4(row, k, K, vec), load4(row, k + 4, K, vec)));
#pragma unroll
  for (int d = T; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
  if ((tid & 63) < T) part[tid >> 6][r] = most;
  __syncthreads();
  most = part[0][r];
#pragma unroll
  for (int w = 1; w < 16; ++w) most = fmaxf(most, part[w][r]);
  const unsigned sb = scale_to(most, 13);
  if (unit == 0) inv[m] = 512.0f * inverse_scale(sb);
  half8 *dst = pieces + (long)(m >> 4) * steps * 128 + (m & 15);
  for (int i = unit; i < steps * 4; i += 1024 / T) {  // eight channels: step i / 4, quarter i % 4
    if (i != unit) {
      u = load4(row, 8 * i, K, vec);
      v = load4(row, 8 * i + 4, K, vec);
    }
    half4v h[2]{}, l[2]{};
    if (m < M) {
      split4(u, __uint_as_float(sb), &h[0], &l[0]);
      split4(v, __uint_as_float(sb), &h[1], &l[1]);
    }
    half8 *at = dst + (long)(i >> 2) * 128 + (i & 3) * 16;
    at[0] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
    at[64] = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// 5 to 32 tokens, MT tiles of 16. A wave takes NT row tiles of the weight and all
// tokens over a range of K blocks; the waves of a workgroup are wk ranges x runs of
// tiles. Codes and pieces come straight from memory, a block of codes and a step
// of pieces ahead. Bound: latency and the pieces' reads from L2 (each workgroup
// reads all tokens), which NT tiles a wave share. With the pieces' launch: 16
// tokens, 4096 x 4096 9.7 us, 2560 x 2048 7.3 us; 32 tokens 14.8 and 9.9 us.
template <int PT, int GPB, int MT, int NT>
__global__ __launch_bounds__(512) void q4_few_kernel(const Q4LinearArgs a) {
  constexpr int SPG = 4 / GPB;
  extern __shared__ __attribute__((aligned(16))) float red[];  // [wave][MT * NT][4][64]
  const Factors factors;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % a.wk, wn = wave / a.wk;
  const int row = lane & 15, quarter = lane >> 4;
  const int runs = (int)(blockDim.x >> 6) / a.wk;
  const long tile0 = ((long)blockIdx.x * runs + wn) * NT;
  const int b0 = wk * a.blocks_per_wave, b1 = min(a.blocks, b0 + a.blocks_per_wave);
  const char *codes[NT], *params[NT];
  tile_addresses<PT, GPB, NT>(a, tile0, lane, codes, params);
  const half8 *xp = reinterpret_cast<const half8 *>(a.pieces) + lane;
  const long pitch = (long)a.blocks * 512;  // a token tile's pieces

  f32x4 acc[MT][NT], sum[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  BlockWeights<PT, GPB, NT> w[2];
  half8 hi[2][MT], lo[2][MT];
  auto load_x = [&](int step, int slot) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      hi[slot][i] = xp[i * pitch + (long)step * 128];
      lo[slot][i] = xp[i * pitch + (long)step * 128 + 64];
    }
  };
  if (b0 < b1) {
    load_x(4 * b0, 0);
    w[0].load(codes, params, b0);
  }
  for (int b = b0; b < b1; ++b) {
    w[1].load(codes, params, min(b + 1, b1 - 1));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      load_x(min(4 * b + j + 1, 4 * b1 - 1), (j + 1) & 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const half8 wf = weights8(w[0].w[t][j], w[0].p[t].zero(j / SPG), factors);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (j % SPG == 0) sum[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
          sum[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[j & 1][i], wf, sum[i][t], 0, 0, 0);
          sum[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[j & 1][i], wf, sum[i][t], 0, 0, 0);
        }
        if (j % SPG == SPG - 1) {
          const float s = w[0].p[t].scale(j / SPG);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(sum[i][t][e], s, acc[i][t][e]);
        }
      }
    }
    w[0] = w[1];
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[((wave * MT * NT + i * NT + t) * 4 + e) * 64 + lane] = acc[i][t][e];
  __syncthreads();
  // The ranges' sums, in range order, over all threads.
  for (int c = threadIdx.x; c < runs * MT * NT * 256; c += blockDim.x) {
    const int l = c & 63, e = c >> 6 & 3, it = c >> 8;  // lane, element, (run, token tile, row tile)
    const int t = it % NT, i = it / NT % MT, r = it / (NT * MT);
    const long n = (((long)blockIdx.x * runs + r) * NT + t) * 16 + (l & 15);
    const int m = i * 16 + 4 * (l >> 4) + e;
    if (n >= a.N || m >= a.M) continue;
    float v = 0.0f;
    for (int q = 0; q < a.wk; ++q) v += red[(((r * a.wk + q) * MT * NT + i * NT + t) * 4 + e) * 64 + l];
    a.out[(long)m * a.N + n] = fmaf(v, a.inv[m], a.bias ? a.bias[n] : 0.0f);
  }
}

// More tokens: tiles of 32 MT tokens x 64 NT rows of the weight, eight waves (2 x 4)
// of MT x NT products of 16 x 16 each, on one of `splits` ranges of K. The pieces
// of a 128-channel block come straight into LDS (two buffers, the next block's in
// flight), in the order in which they are read; codes go to the registers of the
// wave that widens them, a block ahead. One barrier a block. Groups under 128 take
// NT = 2 with MT = 4: their scales and zeros would not fit the registers.
// Bound: the matrix cores (two instructions a product) beside the widening, which
// a wave does for 16 NT rows and uses MT times, and a scaling FMA an output and group.
// 2048 tokens x 4096 x 4096: 115 us, 1.2 PFLOP/s of binary16 products (a library
// product of 4096 x 4096 binary16 matrices runs at 1.18); 512 tokens 52 us with the
// pieces.
template <int PT, int GPB, int MT, int NT>
__global__ __launch_bounds__(512, 2) void q4_tile_kernel(const Q4LinearArgs a) {
  constexpr int SPG = 4 / GPB, TILE = 2 * MT * 8192;  // bytes of a block's pieces
  __shared__ __attribute__((aligned(16))) char x_lds[2][TILE];
  const Factors factors;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 15, quarter = lane >> 4;
  // Ids equal modulo 8 run on one XCD: each takes a contiguous run of the order,
  // in which the tiles of the same tokens are neighbours.
  int id = blockIdx.x;
  {
    const int g = gridDim.x, q = g >> 3, r = g & 7, xcd = id & 7;
    id = xcd * q + min(xcd, r) + (id >> 3);
  }
  const int nblocks = (a.tiles + 4 * NT - 1) / (4 * NT);
  const int nb = id % nblocks, mb = id / nblocks % a.mblocks, split = id / nblocks / a.mblocks;
  const int wm = wave >> 2, wn = wave & 3;
  const long tile0 = (long)nb * (4 * NT) + wn * NT;
  const int b0 = split * a.blocks_per_wave, b1 = min(a.blocks, b0 + a.blocks_per_wave);
  const char *codes[NT], *params[NT];
  tile_addresses<PT, GPB, NT>(a, tile0, lane, codes, params);

  // 1 KB a wave and copy: 8 of a token tile's block, MT / 2 token tiles of a wave.
  // (Token tiles past the last are read as the last and not stored.)
  // Copies and codes are issued a few at a time: a burst would hold the waves up.
  auto fetch = [&](int b, int part, int parts) {
    const int buf = b & 1;
#pragma unroll
    for (int i = 2 * MT * part / parts; i < 2 * MT * (part + 1) / parts; ++i) {
      const int t = min(mb * 2 * MT + i, a.mtiles - 1);
      const char *src = reinterpret_cast<const char *>(a.pieces) + ((long)t * a.blocks + b) * 8192 + wave * 1024;
      copy16(src, lane * 16, x_lds[buf] + i * 8192 + wave * 1024);
    }
  };
  f32x4 acc[MT][NT], sum[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  BlockWeights<PT, GPB, NT> w, next;
  half8 hi[MT], lo[MT], wf[NT];
  auto read = [&](int buf, int at, half8 (&to)[MT]) {
    const half8 *const xl = reinterpret_cast<const half8 *>(x_lds[buf] + wm * MT * 8192) + lane;
#pragma unroll
    for (int i = 0; i < MT; ++i) to[i] = xl[i * 512 + at * 64];
  };
  fetch(b0, 0, 1);
  w.load(codes, params, b0);
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  if (b0 + 1 < b1) {
    fetch(b0 + 1, 0, 4);
    next.load(codes, params, b0 + 1);
  }
  read(b0 & 1, 1, lo);
#pragma unroll
  for (int t = 0; t < NT; ++t) wf[t] = weights8(w.w[t][0], w.p[t].zero(0), factors);
  // Beside a tile's matrix instructions stand the vector ones of the tile before:
  // its scaling, and its weights of the next 32 channels.
  for (int b = b0; b < b1; ++b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      read(b & 1, 2 * j, hi);
      if (j < 2 && b + 1 < b1) fetch(b + 1, 2 * j + 1, 4);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (j % SPG == 0) sum[i][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
          sum[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[i], wf[t], sum[i][t], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
      if (j < 3) {
        read(b & 1, 2 * j + 3, lo);
        if (j == 0 && b + 1 < b1) fetch(b + 1, 2, 4);
        if (j == 1 && b > b0 && b + 1 < b1) next.load(codes, params, b + 1);
      } else {
        // This block's pieces are all in registers, the next block's in LDS.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        next.here();  // (the compiler would wait at their first use, for the copies below too)
        if (b + 2 < b1) fetch(b + 2, 0, 4);
        if (b + 1 < b1) read((b + 1) & 1, 1, lo);
      }
#pragma unroll
      for (int t = 0; t <= NT; ++t) {
        if (t < NT)
#pragma unroll
          for (int i = 0; i < MT; ++i)
            sum[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[i], wf[t], sum[i][t], 0, 0, 0);
        if (t > 0) {
          if (j % SPG == SPG - 1) {
            const float s = w.p[t - 1].scale(j / SPG);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][t - 1][e] = fmaf(sum[i][t - 1][e], s, acc[i][t - 1][e]);
          }
          wf[t - 1] = j < 3 ? weights8(w.w[t - 1][j < 3 ? j + 1 : 0], w.p[t - 1].zero((j < 3 ? j + 1 : 0) / SPG), factors)
                            : weights8(next.w[t - 1][0], next.p[t - 1].zero(0), factors);
        }
        if (t > 0 && t < NT)
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    w = next;
  }
  const bool part = a.splits > 1;
  float *const out = part ? a.partial + (long)split * a.M * a.N : a.out;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const long n = (tile0 + t) * 16 + row;
    if (n >= a.N) continue;
    const float bias = a.bias && !part ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long m = (long)(mb * 2 * MT + wm * MT + i) * 16 + 4 * quarter + e;
        if (m < a.M) out[m * a.N + n] = part ? acc[i][t][e] : fmaf(acc[i][t][e], a.inv[m], bias);
      }
  }
}

// out = (the ranges' partial sums, in range order) / the token's scale + bias.
__global__ __launch_bounds__(256) void q4_reduce_kernel(const Q4LinearArgs a) {
  const long n = (long)blockIdx.x * 256 + threadIdx.x, m = blockIdx.y, stride = (long)a.M * a.N;
  if (n >= a.N) return;
  const float *p = a.partial + m * a.N + n;
  float v = 0.0f;
  for (int s = 0; s < a.splits; ++s) v += p[s * stride];
  a.out[m * a.N + n] = fmaf(v, a.inv[m], a.bias ? a.bias[n] : 0.0f);
}

namespace {

template <int PT, int GPB, int MT, int NT>
hipError_t few_n(hipStream_t st, Q4LinearArgs a) {
  const int groups = (a.tiles + NT - 1) / NT;
  a.wk = 1;
  while (a.wk < 8 && 2 * a.wk <= a.blocks && (long)groups * a.wk < 2048) a.wk *= 2;
  a.blocks_per_wave = (a.blocks + a.wk - 1) / a.wk;
  const int runs = 8 / a.wk;
  const dim3 grid((unsigned)((groups + runs - 1) / runs));
  hipLaunchKernelGGL((q4_few_kernel<PT, GPB, MT, NT>), grid, dim3(512), 8 * MT * NT * 1024, st, a);
  return hipGetLastError();
}
template <int PT, int GPB, int MT>
hipError_t few(hipStream_t st, const Q4LinearArgs &a) {
  // (One row tile a wave while that leaves a CU without a workgroup: 16 tokens,
  // 4096 x 4096 9.4 us against 11.4 with two; 8192 x 4096 15.3 against 13.6; 32
  // tokens, 14336 x 4096 34 against 23.)
  return a.tiles < 2 * 256 ? few_n<PT, GPB, MT, 1>(st, a) : few_n<PT, GPB, MT, 2>(st, a);
}

template <int PT, int GPB, int MT, int NT>
hipError_t tile(hipStream_t st, Q4LinearArgs a) {
  a.mblocks = (a.mtiles + 2 * MT - 1) / (2 * MT);
  const long grid = (long)a.mblocks * ((a.tiles + 4 * NT - 1) / (4 * NT)) * a.splits;
  hipLaunchKernelGGL((q4_tile_kernel<PT, GPB, MT, NT>), dim3((unsigned)grid), dim3(512), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(q4_reduce_kernel, dim3((unsigned)((a.N + 255) / 256), (unsigned)a.M), dim3(256), 0, st, a);
  return hipGetLastError();
}

// Whether tokens are few: up to 32, or 16 where K is past 8192 (each workgroup reads all
// pieces, which its few rows do not repay). us, few and tiles: 32
// tokens, 4096 x 4096 14.8 and 18.0, 14336 x 4096 23 and 31, 4096 x 14336 43 and 34; 16
// of the last 27 and 33; 64, which had twice the tiles a wave, 22 and 21, 35 and 34,
// 62 and 36.
bool q4_few_tokens(long M, long blocks) { return M <= 16 || (M <= 32 && blocks <= 64); }

// Tile shape and ranges of K of a projection of more tokens; the larger
// shape is 128 tokens x big_tiles row tiles. It wins once it fills three quarters
// of the CUs (4096 x 4096, groups of 128: 2048 tokens 129 us against 144, 1536
// level at 113, 1024 111 against 79); below, 64 x 8 row tiles, over ranges of K
// while a CU stays without a workgroup (256 tokens: 50 us with one range, 39 with
// two; 512 tokens: 52 and 54).
struct Q4TilePlan {
  bool big;
  int splits;
};
Q4TilePlan q4_tile_plan(long M, long tiles, long blocks, int big_tiles) {
  Q4TilePlan p{};
  const long big = ((M + 127) / 128) * ((tiles + big_tiles - 1) / big_tiles), small = ((M + 63) / 64) * ((tiles + 7) / 8);
  p.big = big >= 192;
  p.splits = p.big ? 1 : (int)std::max<long>(1, std::min(256 / small, blocks / 4));
  while ((p.splits - 1) * ((blocks + p.splits - 1) / p.splits) >= blocks) --p.splits;  // (no range empty)
  return p;
}

template <int PT, int GPB>
hipError_t run(hipStream_t st, Q4LinearArgs a) {
  if (a.M <= 4) {
    // Waves of a workgroup share K: while tiles are few, and up to 8192 waves where the
    // ranges come out even. (One token: 2048 x 8192 5.9 us with up to 16 waves, 8.7
    // with 8; 16384 x 4096 10.0 with eight ranges, 15.7 with two; 65536 x 1152, three
    // rounds, 16.9 with two, 14.4 with one. Four tokens' activations take the LDS of 8;
    // 14336 x 4096 18 us with four ranges, 26 with two.)
    const int rounds = (a.blocks + 3) / 4;
    a.wk = 1;
    const int most = a.M == 1 ? 16 : 8;
    auto even = [&](int wk) { return (rounds + wk - 1) / wk * wk * 4 <= rounds * 5; };
    while (a.wk < most && a.wk < rounds &&
           ((long)a.tiles * a.wk < 2048 || ((long)a.tiles * a.wk < 8192 && even(2 * a.wk))))
      a.wk *= 2;
    // Two row tiles a wave where there are thousands: its activations are split once
    // for both. (262144 x 1152 35 us against 41, 128256 x 2048 29 against 35; 65536 x
    // 1152 level; four spill.)
    const bool two = a.M == 1 && a.tiles >= 6144;
    if (two) a.wk = 1;
    a.blocks_per_wave = ((rounds + a.wk - 1) / a.wk) * 4;
    const int waves = std::max(4, a.wk), runs = waves / a.wk * (two ? 2 : 1);
    const dim3 grid((unsigned)((a.tiles + runs - 1) / runs));
    if (two) hipLaunchKernelGGL((q4_gemv_kernel<PT, GPB, 1, 2>), grid, dim3(waves * 64), 0, st, a);
    else if (a.M == 1) hipLaunchKernelGGL((q4_gemv_kernel<PT, GPB, 1, 1>), grid, dim3(waves * 64), 0, st, a);
    else hipLaunchKernelGGL((q4_gemv_kernel<PT, GPB, 4, 1>), grid, dim3(waves * 64), 0, st, a);
    return hipGetLastError();
  }
  // (2048 tokens x 4096: 8 a workgroup 15.5 us, 1 a workgroup 30; few tokens want the
  // workgroups.)
  const dim3 rows((unsigned)(a.mtiles * (a.M > 64 ? 2 : 16)));
  auto pieces = a.M > 64 ? q4_pieces_kernel<8> : q4_pieces_kernel<1>;
  hipLaunchKernelGGL(pieces, rows, dim3(1024), 0, st, a.x, a.M, a.K, a.blocks * 4, a.vec, (half8 *)a.pieces, (float *)a.inv);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (q4_few_tokens(a.M, a.blocks)) {
    return a.mtiles == 1 ? few<PT, GPB, 1>(st, a) : few<PT, GPB, 2>(st, a);
  } else {
    const Q4TilePlan p = q4_tile_plan(a.M, a.tiles, a.blocks, GPB == 1 ? 16 : 8);
    a.splits = p.splits;
    a.blocks_per_wave = (a.blocks + p.splits - 1) / p.splits;
    return p.big ? tile<PT, GPB, 4, GPB == 1 ? 4 : 2>(st, a) : tile<PT, GPB, 2, 2>(st, a);
  }
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

// The workspace: pieces, inverse scales, and the partial sums of split K (0 bytes: none).
size_t q4_linear_workspace(long M, long N, long tiles, long blocks, int pack_group) {
  if (M <= 4) return 0;
  const size_t mt = (size_t)(M + 15) / 16;
  const int splits = q4_few_tokens(M, blocks) ? 1 : q4_tile_plan(M, tiles, blocks, pack_group == 128 ? 16 : 8).splits;
  return mt * blocks * 8192 + mt * 16 * sizeof(float) + (splits > 1 ? (size_t)splits * M * N * sizeof(float) : 0);
}

hipError_t launch_q4_linear(hipStream_t st, const Q4LinearArgs &base, int group, int param_type, void *workspace) {
  Q4LinearArgs a = base;
  a.mtiles = (a.M + 15) / 16;
  a.vec = a.K % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  if (workspace) {
    a.pieces = workspace;
    a.inv = reinterpret_cast<const float *>(static_cast<char *>(workspace) + (size_t)a.mtiles * a.blocks * 8192);
    a.partial = const_cast<float *>(a.inv) + a.mtiles * 16;
  }
  switch (param_type) {
    case 0: return run_g<0>(st, a, group);
    case 1: return run_g<1>(st, a, group);
    case 2: return run_g<2>(st, a, group);
    case 3: return run_g<3>(st, a, group);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace spissa
