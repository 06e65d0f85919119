// q4_chunk.hip -- attention of several queries over a KV cache held in 4 bits
// (q4_cache.hip has the format), on v_mfma_f32_16x16x32_f16 with f32 sums.
//
// The products are f32's in all but name. Scores: a code is a whole number and
// so exact in binary16; the queries, scaled by a power of two that takes their
// row's largest to 2^9..2^10, are two binary16 pieces (22 bits). A 32-channel
// group is the depth of one instruction, so its product is scaled by the key's
// step in f32, and the minima times the queries' group sums (three pieces) are
// one more instruction over the groups:
//   s = 2^-e (sum_g step_g (code . q)_g + sum_g min_g (sum q)_g).
// Output: the values, step * code + min scaled by a power of two from the
// head's largest, and the probabilities, times 2^6, are two pieces each, of
// whose four products the three above 2^-22 are taken.
//
// A workgroup (four waves) takes 64 QT rows of a KV head, a row being a (query,
// query head of the group) pair with the head fastest, so that short chunks
// fill the instruction's 16 columns with heads. Per tile of BN keys it widens
// the codes into LDS once for all of them: the keys as they are, in the order in
// which lanes take the A operand, the values as two pieces of V^T. The scores
// are formed as S^T = K Q^T, so a lane has one row (column lane % 16) and four
// keys of each 16, and two such blocks are the B operand of O^T += V^T P^T
// without an exchange, the values' keys being stored in that order.
#include <algorithm>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(2))) _Float16 half2v;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

__device__ __forceinline__ float half_lo(unsigned w) { return (float)__builtin_bit_cast(_Float16, (unsigned short)w); }
__device__ __forceinline__ float half_hi(unsigned w) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
}
// Truncation, two at a time: the second piece takes what the first leaves.
__device__ __forceinline__ half2v pieces2(float a, float b) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// (minus_one: -1 as the compiler does not know it, so that the difference is one
// mixed-precision FMA and not a conversion and a subtraction)
__device__ __forceinline__ void split8(const float (&v)[8], float minus_one, half8 *hi, half8 *lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const half2v h = pieces2(v[2 * i], v[2 * i + 1]);
    const half2v l = pieces2(fmaf((float)h.x, minus_one, v[2 * i]), fmaf((float)h.y, minus_one, v[2 * i + 1]));
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

// A key row's eight codes of a word in the order in which weights of a pair
// come off it: 0, 4, 1, 5, 2, 6, 3, 7 (queries are put in that order too).
// (base: 0x64006400, 1024 twice, in a register: an and-or takes one constant)
__device__ __forceinline__ half8 codes8h(unsigned w, unsigned base) {
  half8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const half2v p = __builtin_bit_cast(half2v, ((w >> (4 * i)) & 0x000f000fu) | base) -
                     (half2v){(_Float16)1024.0f, (_Float16)1024.0f};
    r[2 * i] = p.x;
    r[2 * i + 1] = p.y;
  }
  return r;
}

}  // namespace

template <int D, int QT, int BN>
__global__ __launch_bounds__(256, 2) void q4_chunk_kernel(const Q4ChunkArgs a) {
  constexpr int G = D / 32, DT = D / 16, KT = BN / 16, VB = BN / 32;
  constexpr int DPT = D * BN / 2048;  // channels of a thread's eight keys
  static_assert(DPT == 2 || DPT == 4, "");
  __shared__ __attribute__((aligned(16))) half8 k_lds[KT * G * 64];
  __shared__ __attribute__((aligned(16))) half8 v_lds[2][VB * DT * 64];
  __shared__ __attribute__((aligned(16))) float step_lds[KT * G * 16];
  __shared__ __attribute__((aligned(16))) _Float16 min_lds[BN][8];
  constexpr int CB = BN * D / 2, PB = BN * G * 4, RAW = 2 * (CB + PB);  // bytes of a tile's codes and params
  __shared__ __attribute__((aligned(16))) char raw_lds[RAW];

  float minus_one = -1.0f;
  unsigned base1024 = 0x64006400u;
  asm volatile("" : "+s"(minus_one));
  asm volatile("" : "+v"(base1024));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kq = lane >> 4;
  // Blocks of rows, the last (longest) first; key splits of each.
  const int h = blockIdx.y, split = blockIdx.z;
  const int block = gridDim.x - 1 - blockIdx.x;
  const int rows = a.S * a.R;
  const int row0 = block * (64 * QT) + wave * (16 * QT);
  const int P = a.len - a.S;  // the first query's position
  // keys that any row of the workgroup sees
  const int first_q = block * (64 * QT) / a.R, last_q = min(rows - 1, block * (64 * QT) + 64 * QT - 1) / a.R;
  const int hi = a.causal ? P + last_q + 1 : a.len;
  const int lo = a.window > 0 ? max(0, P + first_q + 1 - a.window) : 0;
  const int t0 = lo / BN + split * a.tps;
  const int t1 = min((hi + BN - 1) / BN, t0 + a.tps);

  // A lane's row, for each of its QT column tiles.
  int pos[QT];
  auto query_row = [&](int t) {  // query * Hq + head
    const int r = min(row0 + 16 * t + col, rows - 1), query = r / a.R;
    return (long)query * a.Hq + h * a.R + (r - query * a.R);
  };
  half8 qh[QT][G], ql[QT][G], qs[QT];
  float inv[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    pos[t] = P + min(row0 + 16 * t + col, rows - 1) / a.R;
    const float *src = a.q + query_row(t) * D + 8 * kq;
    float v[G][8], most = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float4 x = *reinterpret_cast<const float4 *>(src + 32 * g), y = *reinterpret_cast<const float4 *>(src + 32 * g + 4);
      const float u[8] = {x.x, y.x, x.y, y.y, x.z, y.z, x.w, y.w};  // channels 0, 4, 1, 5, ...
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[g][i] = u[i] * a.qscale;
        const float m = fabsf(v[g][i]);
        most = fmaxf(most, m <= 3.402823466e38f ? m : 0.0f);
      }
    }
    most = max32(max16(most));
    const unsigned sb = scale_to(most, 9);
    inv[t] = inverse_scale(sb);
    const float scale = __uint_as_float(sb);
    float sums[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[g][i] *= scale;
        sums[g] += v[g][i];
      }
      split8(v[g], minus_one, &qh[t][g], &ql[t][g]);
      sums[g] = sum32(sum16(sums[g]));
    }
    // the sums' three pieces, one for each of the first three quarters of K
    half8 s0, s1, s2;
    float rest[8];
    split8(sums, minus_one, &s0, &s1);
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = (sums[i] - (float)s0[i]) - (float)s1[i];
    {
      half8 unused;
      split8(rest, minus_one, &s2, &unused);
    }
    __builtin_amdgcn_sched_barrier(0);
    const half8 none{};
    qs[t] = kq == 0 ? s0 : kq == 1 ? s1 : kq == 2 ? s2 : none;
  }
  int wave_hi = 0, wave_lo = 0x7fffffff;  // keys that any row of the wave sees
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t;
    if (r < rows) {
      wave_hi = max(wave_hi, a.causal ? P + min(rows - 1, r + 15) / a.R + 1 : a.len);
      wave_lo = min(wave_lo, a.window > 0 ? max(0, P + r / a.R + 1 - a.window) : 0);
    }
  }

  f32x4 o[QT][DT];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = NEG_INF;
    l[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[t][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  // A tile's codes, steps and minima come as they are, straight into LDS (1 KB a
  // wave and instruction), while the tile before is computed. The rows past the
  // last are read too (the buffers end 64 rows later) and may hold anything:
  // their keys are hidden, and their values taken as zeros.
  const long head = (long)h * a.rows.cap;
  const char *src[4] = {reinterpret_cast<const char *>(a.rows.k) + head * (D / 2),
                        reinterpret_cast<const char *>(a.rows.v) + head * (D / 2),
                        reinterpret_cast<const char *>(a.rows.kp + head * G), reinterpret_cast<const char *>(a.rows.vp + head * G)};
  auto fetch = [&](int tile) {
#pragma unroll
    for (int i = 0; i < (RAW + 4095) / 4096; ++i) {
      const int at = i * 4096 + wave * 1024 + lane * 16;  // raw_lds: keys' codes, values' codes, keys' params, values' params
      if (at >= RAW) continue;
      const int part = at < CB ? 0 : at < 2 * CB ? 1 : at < 2 * CB + PB ? 2 : 3;
      const int off = at - (part == 0 ? 0 : part == 1 ? CB : part == 2 ? 2 * CB : 2 * CB + PB);
      const char *from = part == 0 ? src[0] : part == 1 ? src[1] : part == 2 ? src[2] : src[3];
      __builtin_amdgcn_global_load_lds(from + (long)tile * (part < 2 ? CB : PB) + off,
                                       (__attribute__((address_space(3))) void *)(raw_lds + i * 4096 + wave * 1024), 16, 0, 0);
    }
  };
  const unsigned vsb = scale_to(a.rows.vmax[h], 13);
  const float vscale = __uint_as_float(vsb);

  // A thread's share of a tile: a key's group of 32 channels, and eight keys of
  // DPT channels of the values (keys 4 q + 0..3 and 16 + 4 q + 0..3 of 32).
  constexpr int DC = D / DPT;
  const int kkey = (tid & 15) + 16 * (tid / (16 * G)), kg = (tid >> 4) % G;
  const bool kwork = BN * G >= 256 || tid < BN * G;
  const int vd = tid % DC * DPT, vq = tid / DC % 4, vb = tid / (4 * DC);
  auto widen = [&](int tile) {
    if (kwork) {
      const int kt = kkey >> 4;
      const u32x4 kw = *reinterpret_cast<const u32x4 *>(raw_lds + (kkey * G + kg) * 16);
      const unsigned kp = *reinterpret_cast<const unsigned *>(raw_lds + 2 * CB + (kkey * G + kg) * 4);
#pragma unroll
      for (int q = 0; q < 4; ++q) k_lds[(kt * G + kg) * 64 + q * 16 + (kkey & 15)] = codes8h(kw[q], base1024);
      step_lds[(kt * G + kg) * 16 + (kkey & 15)] = half_lo(kp);
      min_lds[kkey][kg] = __builtin_bit_cast(_Float16, (unsigned short)(kp >> 16));
    }
    float st[8], mn[8];
    unsigned vw[8];
    const char *const params = raw_lds + 2 * CB + PB + ((32 * vb + 4 * vq) * G + vd / 32) * 4;
    const char *const codes = raw_lds + CB + (32 * vb + 4 * vq) * (D / 2) + vd / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned p = *reinterpret_cast<const unsigned *>(params + ((i & 3) + 16 * (i >> 2)) * (G * 4));
      const char *c = codes + ((i & 3) + 16 * (i >> 2)) * (D / 2);
      if constexpr (DPT == 4) vw[i] = *reinterpret_cast<const unsigned short *>(c);
      else vw[i] = *reinterpret_cast<const unsigned char *>(c);
      st[i] = half_lo(p) * vscale;
      mn[i] = half_hi(p) * vscale;
    }
    if ((tile + 1) * BN > a.len) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (tile * BN + 32 * vb + 4 * vq + (i & 3) + 16 * (i >> 2) >= a.len) st[i] = mn[i] = 0.0f;
    }
    const int dt = vd >> 4;
#pragma unroll
    for (int j = 0; j < DPT; ++j) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(st[i], (float)((vw[i] >> (4 * j)) & 15u), mn[i]);
      half8 vh, vl;
      split8(v, minus_one, &vh, &vl);
      // (the low bits mixed with the channel tile: the writes of a wave fall on all banks)
      const int at = (vb * DT + dt) * 64 + ((vq * 16 + (vd & 15) + j) ^ (dt & 7));
      v_lds[0][at] = vh;
      v_lds[1][at] = vl;
    }
  };
  if (G < 8 && tid < BN) {
#pragma unroll
    for (int g = G; g < 8; ++g) min_lds[tid][g] = (_Float16)0.0f;
  }

  if (t0 < t1) fetch(t0);
  for (int tile = t0; tile < t1; ++tile) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a wave's part of the tile is in LDS)
    __syncthreads();  // the tile before is no longer read
    widen(tile);
    __syncthreads();
    if (tile + 1 < t1) fetch(tile + 1);
    const int base = tile * BN;
    // 32 keys at a time: their scores, the rows' maximum, the weights, the output.
#pragma unroll 1
    for (int b = 0; b < VB; ++b) {
      const int key0 = base + 32 * b;
      if (key0 >= wave_hi || key0 + 32 <= wave_lo) continue;
      f32x4 s[2][QT];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const half8 mf = *reinterpret_cast<const half8 *>(min_lds[32 * b + 16 * k + col]);
#pragma unroll
        for (int t = 0; t < QT; ++t)
          s[k][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(mf, qs[t], (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        // two groups' instructions side by side: those that depend on each
        // other are 2 QT apart
#pragma unroll
        for (int g = 0; g < G; g += 2) {
          half8 kf[2];
          f32x4 st[2], c[2][QT];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            kf[i] = k_lds[((2 * b + k) * G + g + i) * 64 + lane];
            st[i] = *reinterpret_cast<const f32x4 *>(&step_lds[((2 * b + k) * G + g + i) * 16 + 4 * kq]);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              c[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], ql[t][g + i], (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < QT; ++t) c[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qh[t][g + i], c[i][t], 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[k][t][e] = fmaf(st[i][e], c[i][t][e], s[k][t][e]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      half8 ph[QT], pl[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        // (32 keys that every row sees need no mask: uniform over the wave)
        const int r = row0 + 16 * t;
        const bool whole = r + 15 < rows && key0 + 32 <= (a.causal ? P + r / a.R + 1 : a.len) &&
                           key0 >= (a.window > 0 ? P + (r + 15) / a.R + 1 - a.window : 0);
        if (!whole) {
          const int kend = r + col < rows ? (a.causal ? pos[t] + 1 : a.len) : 0;
          const int kbeg = a.window > 0 ? pos[t] + 1 - a.window : 0;
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = key0 + 16 * k + 4 * kq + e;
              if (key >= kend || key < kbeg) s[k][t][e] = NEG_INF;
            }
        }
        float top = NEG_INF;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, s[k][t][e]);
        top = max32(max16(top)) * inv[t];
        // The reference rises when a score passes it by 8: weights stay below
        // 2^14, and the output is rarely scaled anew.
        if (__any(top > m[t] + 8.0f)) {
          const float mnew = fmaxf(m[t], top);
          const float alpha = fast_exp2(m[t] - safe_max(mnew));
          m[t] = mnew;
          l[t] *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][d][e] *= alpha;
        }
        const float shift = 6.0f - safe_max(m[t]);
        float p[8];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[4 * k + e] = fast_exp2(fmaf(s[k][t][e], inv[t], shift));
            l[t] += p[4 * k + e];
          }
        split8(p, minus_one, &ph[t], &pl[t]);
      }
      __builtin_amdgcn_sched_barrier(0);
      // two channel tiles side by side, for the same reason
#pragma unroll
      for (int d = 0; d < DT; d += 2) {
        half8 vh[2], vl[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          vh[i] = v_lds[0][(b * DT + d + i) * 64 + (lane ^ ((d + i) & 7))];
          vl[i] = v_lds[1][(b * DT + d + i) * 64 + (lane ^ ((d + i) & 7))];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < QT; ++t) o[t][d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[i], ph[t], o[t][d + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < QT; ++t) o[t][d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[i], pl[t], o[t][d + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < QT; ++t) o[t][d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[i], ph[t], o[t][d + i], 0, 0, 0);
        if (d % 4 == 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  const float vinv = inverse_scale(vsb);
  const long total = (long)a.S * a.Hq;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float sum = sum32(sum16(l[t]));
    const long orow = query_row(t);
    if (row0 + 16 * t + col >= rows) continue;
    float *dst;
    float f;
    if (a.splits > 1) {
      float *ml = a.part_ml + ((long)split * total + orow) * 2;
      if (kq == 0) {
        ml[0] = m[t];
        ml[1] = sum;
      }
      dst = a.part_o + ((long)split * total + orow) * D;
      f = vinv;
    } else {
      if (kq == 0 && !(sum > 0.0f && sum < __builtin_inff())) atomicOr(a.err, kDevErrSoftmaxDenominator);
      dst = a.out + orow * D;
      f = vinv / sum;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<float4 *>(dst + 16 * d + 4 * kq) =
          make_float4(o[t][d][0] * f, o[t][d][1] * f, o[t][d][2] * f, o[t][d][3] * f);
  }
}

namespace {

// Keys of a tile, and column tiles of a wave.
constexpr int chunk_keys(int D) { return D == 256 ? 32 : 64; }
constexpr int chunk_cols(int D) { return D == 256 ? 1 : 2; }

template <int D>
hipError_t chunk(hipStream_t st, const Q4ChunkArgs &a) {
  constexpr int QT = chunk_cols(D), BN = chunk_keys(D);
  const long rows = (long)a.S * a.R;
  const dim3 grid((unsigned)((rows + 64 * QT - 1) / (64 * QT)), (unsigned)a.Hkv, (unsigned)a.splits);
  hipLaunchKernelGGL((q4_chunk_kernel<D, QT, BN>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

Q4ChunkPlan q4_chunk_plan(int D, int S, int R, int Hkv, int len, int causal, int window, int cus) {
  Q4ChunkPlan p;
  const int BN = chunk_keys(D), per = 64 * chunk_cols(D);
  const long blocks = ((long)S * R + per - 1) / per * Hkv;
  // tiles that the workgroup with the most keys visits
  long span = len;
  if (window > 0 && causal) span = std::min<long>(len, (long)window + per / R + 1);
  const long tiles = (span + BN - 1) / BN + 1;
  long splits = std::max<long>(1, 2L * cus / blocks);
  splits = std::min(splits, std::max<long>(1, tiles / 4));
  splits = std::min<long>(splits, 64);
  p.tps = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.tps - 1) / p.tps);
  if (p.splits > 1) p.partial_bytes = (size_t)p.splits * S * R * Hkv * (D + 2) * sizeof(float);
  return p;
}

hipError_t launch_q4_chunk(hipStream_t st, const Q4ChunkArgs &a, int D) {
  switch (D) {
    case 64: return chunk<64>(st, a);
    case 128: return chunk<128>(st, a);
    case 256: return chunk<256>(st, a);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace spissa
