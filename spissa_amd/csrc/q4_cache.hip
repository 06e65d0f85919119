// q4_cache.hip -- the KV cache held in 4 bits: rows in, rows back in f32, and
// the attention of single queries over it.
//
// Format. Of each token and KV head, every 32 channels of a key (or value) row
// have a minimum and a step of their own, both binary16:
//   min = half(lo), step = half((hi - lo) * (1/15)),
//   code = clamp(rne((x - min) * (1 / step)), 0, 15)   (0 where step is 0),
//   value = min + step * code   (the product is exact in f32),
// every operation in f32 and rounded by itself. The minimum takes the channels'
// common offset (which keys have), so the 16 levels span what the 32 channels
// differ by; 32 is the depth of one matrix instruction, and costs 1 bit a
// channel for step and minimum: 0.625 bytes a channel against four.
// HBM layout, keys and values alike: codes [Hkv][cap][D / 2], channel 2 i in
// the low half of byte i; step and minimum [Hkv][cap][D / 32] as one word
// (step in the low half). A head's rows are contiguous, so a head's keys
// stream in whole cache lines, and a row is appended by whole bytes.
#include <algorithm>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

__device__ __forceinline__ float half_lo(unsigned w) { return (float)__builtin_bit_cast(_Float16, (unsigned short)w); }
__device__ __forceinline__ float half_hi(unsigned w) {
  return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
}
__device__ __forceinline__ unsigned half_bits(float v) {
  return __builtin_bit_cast(unsigned short, (_Float16)v);
}

// The eight codes of a word as floats, in channel order.
__device__ __forceinline__ void codes8(unsigned w, float (&c)[8]) {
  const unsigned lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[2 * i] = (float)((lo >> (8 * i)) & 0xffu);
    c[2 * i + 1] = (float)((hi >> (8 * i)) & 0xffu);
  }
}

// All-reduce over aligned groups of eight lanes.
__device__ __forceinline__ float max8(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  return fmaxf(v, dpp<0x141>(v));
}
__device__ __forceinline__ float min8(float v) { return -max8(-v); }

constexpr float kHalfMax = 65504.0f;

// Eight lanes' 32 channels, four each, into codes; lane 0 of the eight stores
// their step and minimum. Returns the largest |value| that the codes can stand for.
__device__ __forceinline__ float hold32(const float4 x, bool store, bool first, unsigned char *codes, unsigned *param,
                                        bool *bad) {
#pragma clang fp contract(off)
  const float v[4] = {x.x, x.y, x.z, x.w};
  float lo = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
  float hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
#pragma unroll
  for (int i = 0; i < 4; ++i) *bad = *bad || !(fabsf(v[i]) <= kHalfMax);
  // (what is not finite is reported, and held as something finite)
  lo = fminf(fmaxf(min8(lo), -kHalfMax), kHalfMax);
  hi = fminf(fmaxf(max8(hi), -kHalfMax), kHalfMax);
  // The step is rounded to f32 and then to binary16: the barrier keeps the
  // product and the conversion from becoming one mixed-precision instruction,
  // which rounds once (one step in some thousands came out a place apart).
  float width = (hi - lo) * (1.0f / 15.0f);
  asm volatile("" : "+v"(width));
  const unsigned mb = half_bits(lo), sb = half_bits(width);
  const float min = half_lo(mb), step = half_lo(sb);
  const float inv = step > 0.0f ? 1.0f / step : 0.0f;
  unsigned c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = fminf(fmaxf(rintf((v[i] - min) * inv), 0.0f), 15.0f);
    c |= (unsigned)t << (4 * i);
  }
  if (store) {
    *reinterpret_cast<unsigned short *>(codes) = (unsigned short)c;
    if (first) *param = mb << 16 | sb;
  }
  return fmaxf(fabsf(min), fabsf(min + 15.0f * step));
}

}  // namespace

// Appends the rows of S tokens of each sequence (blockIdx.z): keys QK-normed
// and rotated, values as they are; with Hq > 0 the query rows too, normed,
// rotated and prescaled into q_out. A row is spread over D/8 lanes, each with
// channels [4 s, 4 s + 4) and [D/2 + 4 s, ...): rotate-half partners, and eight
// consecutive lanes hold 32 consecutive channels of either half.
// Bound: HBM (reads 8 bytes and writes 1.25 for a channel of K and V).
template <int D>
__global__ __launch_bounds__(256) void q4_append_kernel(const Q4AppendArgs a) {
  constexpr int LPR = D / 8, RPW = 64 / LPR, HALF = D / 2;
  const int b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane % LPR;
  const int per = a.Hq + 2 * a.Hkv, total = a.S * per;
  const int row = (blockIdx.x * 4 + wave) * RPW + lane / LPR;
  const bool live = row < total;
  const int at = live ? row : total - 1;
  const int tok = at / per, slot = at - tok * per;
  const bool is_q = slot < a.Hq, is_v = slot >= a.Hq + a.Hkv;
  const int h = is_q ? slot : is_v ? slot - a.Hq - a.Hkv : slot - a.Hq;
  const long t = (long)b * a.S + tok;
  const Q4Rows &seq = a.seq[b];
  const int pos = seq.first + tok;

  const float *src = is_q ? a.q + (t * a.Hq + h) * D : (is_v ? a.v : a.k) + (t * a.Hkv + h) * D;
  float4 x0 = *reinterpret_cast<const float4 *>(src + 4 * sub);
  float4 x1 = *reinterpret_cast<const float4 *>(src + HALF + 4 * sub);
  {
#pragma clang fp contract(off)
    if (a.q_norm) {
      float ss = (x0.x * x0.x + x0.y * x0.y) + (x0.z * x0.z + x0.w * x0.w);
      ss += (x1.x * x1.x + x1.y * x1.y) + (x1.z * x1.z + x1.w * x1.w);
      ss = group_sum<LPR>(ss);
      const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
      const float *nw = is_q ? a.q_norm : a.k_norm;
      const float4 w0 = *reinterpret_cast<const float4 *>(nw + 4 * sub);
      const float4 w1 = *reinterpret_cast<const float4 *>(nw + HALF + 4 * sub);
      if (!is_v) {
        x0 = make_float4(x0.x * inv * w0.x, x0.y * inv * w0.y, x0.z * inv * w0.z, x0.w * inv * w0.w);
        x1 = make_float4(x1.x * inv * w1.x, x1.y * inv * w1.y, x1.z * inv * w1.z, x1.w * inv * w1.w);
      }
    }
    if (a.cos && !is_v) {
      const float4 c = *reinterpret_cast<const float4 *>(a.cos + (long)pos * HALF + 4 * sub);
      const float4 s = *reinterpret_cast<const float4 *>(a.sin + (long)pos * HALF + 4 * sub);
      rotate_pair(x0.x, x1.x, c.x, s.x);
      rotate_pair(x0.y, x1.y, c.y, s.y);
      rotate_pair(x0.z, x1.z, c.z, s.z);
      rotate_pair(x0.w, x1.w, c.w, s.w);
    }
    if (a.q_norm && is_q) {
      x0 = make_float4(x0.x * a.prescale, x0.y * a.prescale, x0.z * a.prescale, x0.w * a.prescale);
      x1 = make_float4(x1.x * a.prescale, x1.y * a.prescale, x1.z * a.prescale, x1.w * a.prescale);
    }
  }
  if (is_q && live) {
    float *dst = a.q_out + (t * a.Hq + h) * D;
    *reinterpret_cast<float4 *>(dst + 4 * sub) = x0;
    *reinterpret_cast<float4 *>(dst + HALF + 4 * sub) = x1;
  }
  // (every lane takes part in the exchanges; query rows and lanes past the last row store nothing)
  const long at_row = (long)h * seq.cap + pos;
  unsigned char *codes = (is_v ? seq.v : seq.k) + at_row * (D / 2);
  unsigned *param = (is_v ? seq.vp : seq.kp) + at_row * (D / 32);
  const bool keep = live && !is_q;
  bool bad = false;
  float big = hold32(x0, keep, (sub & 7) == 0, codes + 2 * sub, param + sub / 8, &bad);
  big = fmaxf(big, hold32(x1, keep, (sub & 7) == 0, codes + HALF / 2 + 2 * sub, param + D / 64 + sub / 8, &bad));
  if (keep && bad) atomicOr(a.err, kDevErrCacheValue);
  // The head's largest |value| (a bound: it never shrinks), which scales the
  // 16-bit pieces of the chunk attention's values. Positive floats order as integers.
  big = max8(big);
  if constexpr (LPR >= 16) big = fmaxf(big, dpp<0x140>(big));
  if constexpr (LPR >= 32) big = max16(big);
  if (keep && is_v && sub == 0 && big > seq.vmax[h])
    atomicMax(reinterpret_cast<int *>(seq.vmax + h), __float_as_int(big));
}

// Rows [first, first + n) of a cache as the f32 values they stand for, keys
// and values [n, Hkv, D]; a thread takes eight channels. Bound: HBM.
__global__ __launch_bounds__(256) void q4_rows_kernel(const Q4Rows s, int n, int Hkv, int D, float *k_out, float *v_out) {
  const int w8 = D / 8;
  const long per = (long)n * Hkv * w8;
  long i = (long)blockIdx.x * 256 + threadIdx.x;
  const bool is_v = blockIdx.y != 0;
  float *out = is_v ? v_out : k_out;
  if (i >= per || !out) return;
  const int c = (int)(i % w8);
  const long th = i / w8;
  const int h = (int)(th % Hkv);
  const long row = (long)h * s.cap + s.first + th / Hkv;
  const unsigned word = reinterpret_cast<const unsigned *>(is_v ? s.v : s.k)[row * w8 + c];
  const unsigned p = (is_v ? s.vp : s.kp)[row * (D / 32) + c / 4];
  const float step = half_lo(p), min = half_hi(p);
  float v[8];
  codes8(word, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = fmaf(step, v[j], min);
  float4 *dst = reinterpret_cast<float4 *>(out + i * 8);
  dst[0] = make_float4(v[0], v[1], v[2], v[3]);
  dst[1] = make_float4(v[4], v[5], v[6], v[7]);
}

namespace {

// The keys that the last token of sequence z sees, [lo, hi).
template <int MB>
__device__ __forceinline__ void visible(const Q4AttnArgsOf<MB> &a, int z, int *lo, int *hi) {
  *hi = a.seq[z].len;
  *lo = a.window > 0 ? max(0, *hi - a.window) : 0;
}

}  // namespace

// One query of RB heads of a KV head (blockIdx.x) over one range of keys
// (blockIdx.y) of sequence blockIdx.z. A row is spread over D/16
// lanes of 16 channels (8 bytes of codes, half a 32-channel group):
//   q.k = step * sum q code + min * sum q   (the lane's part), and
//   o += (p step) code, o_min += p min,
// so a code costs one conversion and one FMA a head, all in f32.
template <int D, int RB, int RPG, int MB>
__global__ __launch_bounds__(256) void q4_attend_kernel(const Q4AttnArgsOf<MB> a) {
  constexpr int LPR = D / 16, GPW = 64 / LPR, NG = 4 * GPW, ENTRY = RB * (D + 2);
  __shared__ float red_o[4][RB][D];
  __shared__ float red_l[4][RB], wave_m[4][RB];

  const int z = blockIdx.z, hb = blockIdx.x % a.HB, h = blockIdx.x / a.HB, split = blockIdx.y;
  int lo, hi;
  visible(a, z, &lo, &hi);
  const int k0 = lo + split * a.kps, k1 = min(hi, k0 + a.kps);
  if (k0 >= hi) return;  // (split 0 always has a key: the query's own)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane % LPR, grp = wave * GPW + lane / LPR;
  const Q4Rows &seq_rows = a.seq[z].rows;
  const uint2 *kc = reinterpret_cast<const uint2 *>(seq_rows.k) + (long)h * seq_rows.cap * LPR;
  const uint2 *vc = reinterpret_cast<const uint2 *>(seq_rows.v) + (long)h * seq_rows.cap * LPR;
  const unsigned *kp = seq_rows.kp + (long)h * seq_rows.cap * (D / 32);
  const unsigned *vp = seq_rows.vp + (long)h * seq_rows.cap * (D / 32);

  float q[RB][16], qsum[RB], o[RB][16], omin[RB], m[RB], l[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int head = h * a.R + min(hb * RB + r, a.R - 1);  // (the last block may have heads to spare)
    const float4 *src = reinterpret_cast<const float4 *>(a.q + ((long)z * a.Hq + head) * D + 16 * sub);
    qsum[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 t = src[i];
      q[r][4 * i] = t.x * a.qscale;
      q[r][4 * i + 1] = t.y * a.qscale;
      q[r][4 * i + 2] = t.z * a.qscale;
      q[r][4 * i + 3] = t.w * a.qscale;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      qsum[r] += q[r][i];
      o[r][i] = 0.0f;
    }
    omin[r] = l[r] = 0.0f;
    m[r] = NEG_INF;
  }

  for (int c = k0; c < k1; c += NG * RPG) {
    uint2 kw[RPG], vw[RPG];
    unsigned kpw[RPG], vpw[RPG];
    bool valid[RPG];
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      const int j = c + grp + i * NG;
      valid[i] = j < k1;
      const int jj = valid[i] ? j : k0;  // (a row of the range, its weight 0)
      kw[i] = kc[(long)jj * LPR + sub];
      kpw[i] = kp[(long)jj * (D / 32) + sub / 2];
      vw[i] = vc[(long)jj * LPR + sub];
      vpw[i] = vp[(long)jj * (D / 32) + sub / 2];
    }
    float s[RPG][RB];
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      float e[16];
      codes8(kw[i].x, reinterpret_cast<float(&)[8]>(e[0]));
      codes8(kw[i].y, reinterpret_cast<float(&)[8]>(e[8]));
      const float step = half_lo(kpw[i]), min = half_hi(kpw[i]);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float d = 0.0f;
#pragma unroll
        for (int t = 0; t < 16; ++t) d = fmaf(q[r][t], e[t], d);
        s[i][r] = group_sum<LPR>(fmaf(step, d, min * qsum[r]));
      }
    }
    float alpha[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float top = NEG_INF;
#pragma unroll
      for (int i = 0; i < RPG; ++i) top = valid[i] ? fmaxf(top, s[i][r]) : top;
      if constexpr (LPR <= 4) top = fmaxf(top, dpp<0x124>(top));  // row_ror:4
      top = groups_max<LPR>(top);
      const float mnew = fmaxf(m[r], top), ms = safe_max(mnew);
      alpha[r] = fast_exp2(m[r] - ms);
      m[r] = mnew;
      l[r] *= alpha[r];
      omin[r] *= alpha[r];
#pragma unroll
      for (int t = 0; t < 16; ++t) o[r][t] *= alpha[r];
#pragma unroll
      for (int i = 0; i < RPG; ++i) {
        s[i][r] = valid[i] ? fast_exp2(s[i][r] - ms) : 0.0f;
        l[r] += s[i][r];
      }
    }
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      float e[16];
      codes8(vw[i].x, reinterpret_cast<float(&)[8]>(e[0]));
      codes8(vw[i].y, reinterpret_cast<float(&)[8]>(e[8]));
      const float step = half_lo(vpw[i]), min = half_hi(vpw[i]);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float ps = s[i][r] * step;
        omin[r] = fmaf(s[i][r], min, omin[r]);
#pragma unroll
        for (int t = 0; t < 16; ++t) o[r][t] = fmaf(ps, e[t], o[r][t]);
      }
    }
  }

  // The row groups of a wave share m: their sums add.
  auto add_groups = [&](float v) {
    if constexpr (LPR <= 8) v += dpp0<0x128>(v);  // row_ror:8
    if constexpr (LPR <= 4) v += dpp0<0x124>(v);  // row_ror:4
    return sum32(sum16(v));
  };
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    l[r] = add_groups(l[r]);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const float v = add_groups(o[r][t] + omin[r]);
      if (lane < LPR) red_o[wave][r][16 * sub + t] = v;
    }
    if (lane == 0) {
      red_l[wave][r] = l[r];
      wave_m[wave][r] = m[r];
    }
  }
  __syncthreads();
  const long entry = (((long)z * a.Hkv + h) * a.HB + hb) * a.max_splits + split;
  for (int e = threadIdx.x; e < RB * D; e += 256) {
    const int r = e / D, dim = e % D;
    const float M = fmaxf(fmaxf(wave_m[0][r], wave_m[1][r]), fmaxf(wave_m[2][r], wave_m[3][r]));
    const float Ms = safe_max(M);
    float O = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = fast_exp2(wave_m[w][r] - Ms);
      O = fmaf(red_o[w][r][dim], f, O);
      L = fmaf(red_l[w][r], f, L);
    }
    if (a.max_splits > 1) {
      float *dst = a.partial + entry * (long)ENTRY;
      dst[e] = O;
      if (dim == 0) {
        dst[RB * D + 2 * r] = M;
        dst[RB * D + 2 * r + 1] = L;
      }
    } else if (hb * RB + r < a.R) {
      a.out[((long)z * a.Hq + h * a.R + hb * RB + r) * D + dim] = O / L;
      if (dim == 0 && !(L > 0.0f && L < __builtin_inff())) atomicOr(a.err, kDevErrSoftmaxDenominator);
    }
  }
}

// Merges the key ranges of one (query, KV head, head block). 256 threads: 32
// consecutive outputs x 8 range lanes.
template <int D, int RB, int MB>
__global__ __launch_bounds__(256) void q4_combine_kernel(const Q4AttnArgsOf<MB> a) {
  constexpr int ENTRY = RB * (D + 2), OUTS = 32, SL = 8;
  __shared__ float s_m[SL][OUTS], s_l[SL][OUTS], s_o[SL][OUTS];
  const int z = blockIdx.z, hb = blockIdx.x % a.HB, h = blockIdx.x / a.HB;
  int lo, hi;
  visible(a, z, &lo, &hi);
  const int nsplit = (hi - lo + a.kps - 1) / a.kps;
  const int out = threadIdx.x % OUTS, sl = threadIdx.x / OUTS;
  const int e = blockIdx.y * OUTS + out, r = e / D;
  const float *ents = a.partial + (((long)z * a.Hkv + h) * a.HB + hb) * a.max_splits * (long)ENTRY;
  float m = NEG_INF, l = 0.0f, o = 0.0f;
  for (int s = sl; s < nsplit; s += SL) {
    const float *ent = ents + (long)s * ENTRY;
    const float em = ent[RB * D + 2 * r], el = ent[RB * D + 2 * r + 1], eo = ent[e];
    const float mx = fmaxf(m, em), mxs = safe_max(mx);
    const float f = fast_exp2(m - mxs), g = fast_exp2(em - mxs);
    l = l * f + el * g;
    o = o * f + eo * g;
    m = mx;
  }
  s_m[sl][out] = m;
  s_l[sl][out] = l;
  s_o[sl][out] = o;
  __syncthreads();
  if (sl == 0 && hb * RB + r < a.R) {
    float M = NEG_INF;
#pragma unroll
    for (int k = 0; k < SL; ++k) M = fmaxf(M, s_m[k][out]);
    const float Ms = safe_max(M);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      const float g = fast_exp2(s_m[k][out] - Ms);
      L += s_l[k][out] * g;
      O += s_o[k][out] * g;
    }
    a.out[((long)z * a.Hq + h * a.R + hb * RB) * D + e] = O / L;
    if ((e % D) == 0 && !(L > 0.0f && L < __builtin_inff())) atomicOr(a.err, kDevErrSoftmaxDenominator);
  }
}

namespace {

constexpr int kQ4Rows = 2;  // rows per lane group in flight

template <int D, int RB, int MB>
hipError_t attend(hipStream_t st, const Q4AttnArgsOf<MB> &a, int nz) {
  const dim3 grid((unsigned)(a.Hkv * a.HB), (unsigned)a.max_splits, (unsigned)nz);
  hipLaunchKernelGGL((q4_attend_kernel<D, RB, kQ4Rows, MB>), grid, dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.max_splits == 1) return e;
  const dim3 cgrid((unsigned)(a.Hkv * a.HB), (unsigned)(RB * D / 32), (unsigned)nz);
  hipLaunchKernelGGL((q4_combine_kernel<D, RB, MB>), cgrid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int D, int RB>
hipError_t attend_b(hipStream_t st, const Q4AttnArgs &a, int nz) {
  if (nz == 1) {
    Q4AttnArgsOf<1> one;
    static_cast<Q4AttnBase &>(one) = a;
    one.seq[0] = a.seq[0];
    return attend<D, RB, 1>(st, one, nz);
  }
  return attend<D, RB, kMaxDecodeBatch>(st, a, nz);
}

template <int D>
hipError_t attend_d(hipStream_t st, const Q4AttnArgs &a, int RB, int nz) {
  switch (RB) {
    case 1: return attend_b<D, 1>(st, a, nz);
    case 2: return attend_b<D, 2>(st, a, nz);
    case 3: return attend_b<D, 3>(st, a, nz);
    case 4: return attend_b<D, 4>(st, a, nz);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

bool q4_supported(size_t D) { return D == 64 || D == 128 || D == 256; }

Q4AttnPlan q4_attend_plan(int D, int R, int Hkv, const int *keys, int n) {
  Q4AttnPlan p;
  p.HB = (R + 3) / 4;
  p.RB = (R + p.HB - 1) / p.HB;
  const int chunk = 4 * (64 / (D / 16)) * kQ4Rows;
  long total = 0;
  int most = 1;
  for (int i = 0; i < n; ++i) {
    total += keys[i];
    most = std::max(most, keys[i]);
  }
  const long heads = (long)Hkv * p.HB;
  const long per = (total * heads + kDecodeGridWorkgroups - 1) / kDecodeGridWorkgroups;
  long kps = std::max<long>(1, (per + chunk - 1) / chunk) * chunk;
  if ((most + kps - 1) / kps > kMaxDecodeSplits)
    kps = ((most + kMaxDecodeSplits - 1) / kMaxDecodeSplits + chunk - 1) / chunk * chunk;
  p.kps = (int)kps;
  p.splits = (int)((most + kps - 1) / kps);
  return p;
}

hipError_t launch_q4_attend(hipStream_t st, const Q4AttnArgs &a, int D, int RB, int nz) {
  switch (D) {
    case 64: return attend_d<64>(st, a, RB, nz);
    case 128: return attend_d<128>(st, a, RB, nz);
    case 256: return attend_d<256>(st, a, RB, nz);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_q4_append(hipStream_t st, const Q4AppendArgs &a, int D, int B) {
  const long rows = (long)a.S * (a.Hq + 2 * a.Hkv), per = 4 * (64 / (D / 8));
  const dim3 grid((unsigned)((rows + per - 1) / per), 1, (unsigned)B);
  switch (D) {
    case 64: hipLaunchKernelGGL((q4_append_kernel<64>), grid, dim3(256), 0, st, a); break;
    case 128: hipLaunchKernelGGL((q4_append_kernel<128>), grid, dim3(256), 0, st, a); break;
    case 256: hipLaunchKernelGGL((q4_append_kernel<256>), grid, dim3(256), 0, st, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_q4_rows(hipStream_t st, const Q4Rows &s, size_t n, size_t Hkv, size_t D, float *k_out, float *v_out) {
  const size_t threads = n * Hkv * (D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
  hipLaunchKernelGGL(q4_rows_kernel, grid, dim3(256), 0, st, s, (int)n, (int)Hkv, (int)D, k_out, v_out);
  return hipGetLastError();
}

}  // namespace spissa
