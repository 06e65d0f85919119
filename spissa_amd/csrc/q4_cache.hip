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

__device__ __forceinline__ unsigned half_bits(float v) {
  return __builtin_bit_cast(unsigned short, (_Float16)v);
}

template <int N>
__device__ __forceinline__ void words(const char *p, unsigned (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const unsigned *>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  }
}

// (code - 8) 2^-9 twice. A code in bits 0..3 of a binary16 is code 2^-24, in bits
// 4..7 code 2^-20, so a packed FMA makes it an ordinary number and takes the 8 off.
struct Slots {
  half2v from0, from4, offset;  // (in registers: the compiler does not know them)
  __device__ __forceinline__ Slots() {
    unsigned a = 0x78007800u, b = 0x68006800u, c = 0xa400a400u;  // 2^15, 2^11, -2^-6
    asm volatile("" : "+v"(a), "+v"(b), "+v"(c));
    from0 = __builtin_bit_cast(half2v, a);
    from4 = __builtin_bit_cast(half2v, b);
    offset = __builtin_bit_cast(half2v, c);
  }
  __device__ __forceinline__ half2v low(unsigned w) const {
    return __builtin_elementwise_fma(__builtin_bit_cast(half2v, w & 0x000f000fu), from0, offset);
  }
  __device__ __forceinline__ half2v high(unsigned w) const {
    return __builtin_elementwise_fma(__builtin_bit_cast(half2v, w & 0x00f000f0u), from4, offset);
  }
};
__device__ __forceinline__ half8 join(half2v a, half2v b, half2v c, half2v d) {
  return (half8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// A key word's eight codes as slots: channels 0, 4, 1, 5, 2, 6, 3, 7.
__device__ __forceinline__ half8 code_slots(unsigned w, const Slots &s) {
  return join(s.low(w), s.high(w), s.low(w >> 8), s.high(w >> 8));
}
// The codes of channel n of a lane's CH of eight rows. (The compiler shares what the
// channels of a half word have in common.)
template <int CH, int N>
__device__ __forceinline__ half8 value_slots(const unsigned (&v)[8][N], int n, const Slots &s) {
  half2v r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned w0 = v[2 * i][n / 8], w1 = v[2 * i + 1][n / 8];
    const unsigned u = __builtin_amdgcn_perm(w1, w0, n & 4 ? 0x07060302u : 0x05040100u);
    r[i] = n & 1 ? s.high(n & 2 ? u >> 8 : u) : s.low(n & 2 ? u >> 8 : u);
  }
  return join(r[0], r[1], r[2], r[3]);
}

// The key of 32 in slot i of a lane's eight, above the 4 (lane / 16) that the lanes differ by.
__device__ __forceinline__ constexpr int key_of(int i) { return (i & 3) + 16 * (i >> 2); }

// Over the 16 lanes of a row of them, the sum of the lanes NQ apart: each step leaves
// equal values that many lanes apart, so all lanes add the same pairs.
template <int NQ>
__device__ __forceinline__ float groups_sum(float v) {
  v += dpp0<0x128>(v);                         // row_ror:8
  if constexpr (NQ <= 4) v += dpp0<0x124>(v);  // row_ror:4
  if constexpr (NQ <= 2) v += dpp0<0x122>(v);  // row_ror:2
  return v;
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp<0x128>(v));
  v = fmaxf(v, dpp<0x124>(v));
  v = fmaxf(v, dpp<0x122>(v));
  return fmaxf(v, dpp<0x121>(v));
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
// their step and minimum.
__device__ __forceinline__ void hold32(const float4 x, bool store, bool first, unsigned char *codes, unsigned *param,
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
}

// What a fused step does to query and key rows before they are used or held.
struct RowPrep {
  const float *cos, *sin;        // RoPE table rows by position, or null
  const float *q_norm, *k_norm;  // QK-norm, null: none
  float eps, prescale;
};
// A row over D/8 lanes, of which lane `sub` has channels [4 sub, 4 sub + 4) and
// [D/2 + 4 sub, ...): rotate-half partners, and eight consecutive lanes hold 32
// consecutive channels of either half.
template <int D>
__device__ __forceinline__ void prepare_row(const RowPrep &a, bool is_q, bool is_v, int pos, int sub, float4 &x0, float4 &x1) {
#pragma clang fp contract(off)
  constexpr int HALF = D / 2;
  if (a.q_norm) {
    float ss = (x0.x * x0.x + x0.y * x0.y) + (x0.z * x0.z + x0.w * x0.w);
    ss += (x1.x * x1.x + x1.y * x1.y) + (x1.z * x1.z + x1.w * x1.w);
    ss = group_sum<D / 8>(ss);
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
// ... and into codes: every lane takes part in the exchanges, those with `store`
// write.
template <int D>
__device__ __forceinline__ void hold_row(const float4 &x0, const float4 &x1, int sub, bool store, unsigned char *codes,
                                         unsigned *params, bool *bad) {
  hold32(x0, store, (sub & 7) == 0, codes + 2 * sub, params + sub / 8, bad);
  hold32(x1, store, (sub & 7) == 0, codes + D / 4 + 2 * sub, params + D / 64 + sub / 8, bad);
}

}  // namespace

// Appends the rows of S tokens of each sequence (blockIdx.z): keys QK-normed
// and rotated, values as they are; with Hq > 0 the query rows too, normed,
// rotated and prescaled into q_out.
// Bound: HBM (reads 8 bytes and writes 1.25 for a channel of K and V). 4096 tokens of 8
// heads of 128: 9.5 us, 4.1 TB/s.
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
  prepare_row<D>({a.cos, a.sin, a.q_norm, a.k_norm, a.eps, a.prescale}, is_q, is_v, pos, sub, x0, x1);
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
  hold_row<D>(x0, x1, sub, keep, codes, param, &bad);
  if (keep && bad) atomicOr(a.err, kDevErrCacheValue);
}

// Rows [first, first + n) of a cache as the f32 values they stand for, keys
// and values [n, Hkv, D]; a thread takes eight channels. Bound: HBM (4096 tokens of 8
// heads of 128: 9.4 us, 4.1 TB/s).
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

// (eight waves: a workgroup a CU holds two or three a SIMD)
constexpr int kQ4Waves = 8, kQ4Step = 32 * kQ4Waves;  // waves of a workgroup, and the keys of a step of theirs

// The keys that any of the last S tokens of sequence z sees, [lo, hi).
template <int MB>
__device__ __forceinline__ void visible(const Q4AttnArgsOf<MB> &a, int z, int *lo, int *hi) {
  *hi = a.seq[z].len;
  *lo = a.window > 0 ? max(0, *hi - a.S + 1 - a.window) : 0;
}
// Row r of a KV head h, a (query, head of the group) pair with the head fastest, among
// the rows of the queries and outputs.
template <int MB>
__device__ __forceinline__ long row_of(const Q4AttnArgsOf<MB> &a, int z, int h, int r) {
  if (a.S == 1) return (long)z * a.Hq + h * a.R + r;
  const int query = r / a.R;
  return (long)query * a.Hq + h * a.R + (r - query * a.R);
}

}  // namespace

// NQ rows, heads of a query or of a few, of a KV head (blockIdx.x) over one range of
// keys (blockIdx.y) of sequence blockIdx.z, 32 keys of the range a wave and step.
//
// With G = D / 32 groups a row, the 16 columns of a matrix instruction are NQ =
// 16 / G heads x G groups: column (q, g) of the queries has q's channels of group
// g and zeros elsewhere, so one accumulator gathers sum_g-channels q code for
// every (q, g), and a lane, whose column is one (q, g), adds its group's
//   step * that sum + (min + 8 step) * sum_g q
// for its four keys of 16; the groups' lanes add up to the score. Its weights
// times its group's steps of the values are row (q, g) of the other product
// at once, P' V: a column holds channels of one group, and takes its output from
// that group's rows. (min + 8 step) p goes beside it as one sum a (q, g).
// A lane takes codes in whole words: of a key, the k slots of its quarter are a
// quarter of the row; of the values, a column is D / 16 consecutive channels,
// one a product. Operands are code - 8 (times 2^-9), with min + 8 step beside them:
// with the codes as they are, the sums of many keys' values would grow, and cancel
// against the minima's only at the end (outputs over 8192 keys were 1e-6 off).
// Queries and weights are two nearest binary16 pieces.
// Bound: HBM for many keys, latency (one step of loads, one of sums) for few.
// 16 sequences of 8192 keys, 24 heads on 8 of 128: 40 us, 4.2 TB/s of codes and
// params (a plain read reaches 6.0 to 6.6); 32768 keys of one head of 256: 13 us; 512
// keys, 32 heads on 8 of 64: 6 us. Outputs are 1e-7 off (RMS, relative), where a plain
// f32 form's are 1e-7 to 7e-7.
// STEP: the fused step of one token. Every workgroup prepares its queries and
// holds the sequence's new row of its head in LDS (as q4_append_kernel does, bit for
// bit), and takes that row from there; the one with the last range and the first heads
// writes it. A step over 512 keys, 32 heads on 8 of 64, with its rows read back: 18.2 us
// with a launch of q4_append_kernel before, 14.7 without.
// FEW: several queries of one sequence (S > 1), whose keys end (and begin) at their own.
template <int D, int MB, bool STEP, bool FEW>
__global__ __launch_bounds__(64 * kQ4Waves) void q4_attend_kernel(const Q4AttnArgsOf<MB> a) {
  constexpr int G = D / 32, NQ = 16 / G, CH = D / 16, ENTRY = NQ * (D + 2);
  __shared__ float red_o[kQ4Waves][NQ][D];
  __shared__ float red_l[kQ4Waves][NQ], wave_m[kQ4Waves][NQ];
  __shared__ _Float16 q_lds[2][NQ][D + 8] __attribute__((aligned(16)));
  __shared__ float q_sum[NQ][G], q_inv[NQ];
  static_assert(NQ * D == 64 * kQ4Waves, "a thread a channel of the queries");
  __shared__ __attribute__((aligned(16))) float q_row[STEP ? NQ : 1][D];
  __shared__ __attribute__((aligned(16))) unsigned char new_codes[2][D / 2];
  __shared__ unsigned new_params[2][G];

  const int z = blockIdx.z, hb = blockIdx.x % a.HB, h = blockIdx.x / a.HB, split = blockIdx.y;
  int lo, hi;
  visible(a, z, &lo, &hi);
  const int k0 = lo + split * a.kps, k1 = min(hi, k0 + a.kps);
  if (k0 >= hi) return;  // (split 0 always has a key: the query's own)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, t = lane >> 4, g = col / NQ;
  const Q4Rows &seq_rows = a.seq[z].rows;
  const char *const kc = reinterpret_cast<const char *>(seq_rows.k) + (long)h * seq_rows.cap * (D / 2);
  const char *const vc = reinterpret_cast<const char *>(seq_rows.v) + (long)h * seq_rows.cap * (D / 2);
  const char *const kp = reinterpret_cast<const char *>(seq_rows.kp) + (long)h * seq_rows.cap * (G * 4);
  const char *const vp = reinterpret_cast<const char *>(seq_rows.vp) + (long)h * seq_rows.cap * (G * 4);
  const unsigned k_at = col * (D / 2) + t * (D / 8), v_at = 4 * t * (D / 2) + col * (CH / 2);
  const unsigned p_at = 4 * t * (G * 4) + g * 4;
  const int rows = FEW ? a.S * a.R : a.R;

  // Of 32 keys from c on: two rows' quarters, and of the eight keys 4 t + 0..3 and
  // 16 + 4 t + 0..3 the values' words and both rows' params. (The buffers go on for
  // 128 rows past the last.)
  unsigned kw[2][G], vw[8][CH / 8 + (CH < 8)], kpw[8], vpw[8];
  auto load_k = [&](int c) {
    const char *const rows = kc + (long)c * (D / 2) + k_at, *const params = kp + (long)c * (G * 4) + p_at;
#pragma unroll
    for (int i = 0; i < 2; ++i) words(rows + i * 16 * (D / 2), kw[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) kpw[i] = *reinterpret_cast<const unsigned *>(params + key_of(i) * (G * 4));
  };
  auto load_v = [&](int c) {
    const char *const rows = vc + (long)c * (D / 2) + v_at, *const params = vp + (long)c * (G * 4) + p_at;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      vpw[i] = *reinterpret_cast<const unsigned *>(params + key_of(i) * (G * 4));
      if constexpr (CH < 8) vw[i][0] = *reinterpret_cast<const unsigned short *>(rows + key_of(i) * (D / 2));
      else words(rows + key_of(i) * (D / 2), vw[i]);
    }
  };
  int c = k0 + 32 * wave;
  if (c < k1) {
    load_k(c);
    load_v(c);
  }

  if constexpr (STEP) {
    constexpr int LPR = D / 8;
    const int sub = lane % LPR, r = lane / LPR, pos = hi - 1;
    const RowPrep prep{a.cos, a.sin, a.q_norm, a.k_norm, a.eps, a.prescale};
    if (wave == 0) {  // its 64 lanes are NQ rows
      const float *src = a.q + row_of(a, z, h, min(hb * NQ + r, rows - 1)) * D + 4 * sub;
      float4 x0 = *reinterpret_cast<const float4 *>(src), x1 = *reinterpret_cast<const float4 *>(src + D / 2);
      prepare_row<D>(prep, true, false, pos, sub, x0, x1);
      *reinterpret_cast<float4 *>(&q_row[r][4 * sub]) = x0;
      *reinterpret_cast<float4 *>(&q_row[r][D / 2 + 4 * sub]) = x1;
    } else if (wave == 1) {  // the key and the value
      const bool is_v = r & 1, writes = k1 == hi && hb == 0;
      const float *src = (is_v ? a.v : a.k) + ((long)z * a.Hkv + h) * D + 4 * sub;
      float4 x0 = *reinterpret_cast<const float4 *>(src), x1 = *reinterpret_cast<const float4 *>(src + D / 2);
      prepare_row<D>(prep, false, is_v, pos, sub, x0, x1);
      bool bad = false;
      hold_row<D>(x0, x1, sub, r < 2, new_codes[is_v], new_params[is_v], &bad);
      if (writes && bad) atomicOr(a.err, kDevErrCacheValue);
    }
    __syncthreads();
  }

  // The queries' pieces, a channel a thread, as codes come off a word: 0, 4, 1, 5,
  // 2, 6, 3, 7 of eight. (A head past the last is the last.)
  const int r = threadIdx.x / D, ch = threadIdx.x % D;
  float y;
  if constexpr (STEP) y = q_row[r][ch] * a.qscale;
  else y = a.q[row_of(a, z, h, min(hb * NQ + r, rows - 1)) * D + ch] * a.qscale;
  {
    const float size = fabsf(y);
    const float most = max32(max16(row_max(size <= 3.402823466e38f ? size : 0.0f)));
    if (lane == 0) wave_m[wave][0] = most;
  }
  __syncthreads();
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) most = fmaxf(most, wave_m[r * (D / 64) + i][0]);
  const unsigned sb = scale_to(most, 13);
  y *= __uint_as_float(sb);
  {
    const _Float16 first = (_Float16)y, second = (_Float16)(y - (float)first);
    const int at = (ch & ~7) + (ch & 3) * 2 + (ch >> 2 & 1);
    q_lds[0][r][at] = first;
    q_lds[1][r][at] = second;
    const float sum = group_sum<32>((float)first + (float)second);
    if (ch % 32 == 0) q_sum[r][ch / 32] = sum;
    if (ch == 0) q_inv[r] = inverse_scale(sb);
  }
  __syncthreads();
  half8 qh[G], ql[G];
  // (scores are held as 1 / inv of what they are)
  const float inv = q_inv[col % NQ], qsum = q_sum[col % NQ][g], qsum8 = 8.0f * qsum;
  const Slots slots;
  float minus_one = -1.0f;
  asm volatile("" : "+v"(minus_one));
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int first = t * (D / 4) + 8 * j;
    const half8 none{};
    qh[j] = first / 32 == g ? *reinterpret_cast<const half8 *>(&q_lds[0][col % NQ][first]) : none;
    ql[j] = first / 32 == g ? *reinterpret_cast<const half8 *>(&q_lds[1][col % NQ][first]) : none;
  }
  // FEW: the keys of the column's query, and those that all queries see.
  int row_end = 0, row_begin = 0, all_end = 0, all_begin = 0;
  if constexpr (FEW) {
    const int pos = hi - a.S + min(hb * NQ + col % NQ, rows - 1) / a.R;
    row_end = a.causal ? pos + 1 : hi;
    row_begin = a.window > 0 ? pos + 1 - a.window : 0;
    all_end = a.causal ? hi - a.S + 1 : hi;
    all_begin = a.window > 0 ? hi - a.window : 0;
  }

  f32x4 o[CH];
#pragma unroll
  for (int n = 0; n < CH; ++n) o[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // The weights are scaled by a power of two, a column's own, that their products with
  // its group's steps keep two whole pieces: the largest step so far goes to 2^14..2^15,
  // and one past `cap` moves the scale, as a score past m moves the reference. Beside
  // references past 2^20, whose digits the scale's exponent would be lost in (and the
  // weights overflow), it is 1, which no step is too large for.
  float omin = 0.0f, l = 0.0f, m = NEG_INF, cap = -1.0f;
  unsigned scale = 127u << 23;
  // (no copies of the next step's words: they are asked for when this step's are spent)
  for (; c < k1; c += kQ4Step) {
    const bool more = c + kQ4Step < k1;
    if constexpr (STEP) {
      if (c + 32 >= hi) {  // (the tile has the new row, and k1 is hi)
        const int at = hi - 1 - c;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (16 * i + col == at) words(reinterpret_cast<const char *>(new_codes[0]) + t * (D / 8), kw[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (4 * t + key_of(i) == at) {
            kpw[i] = new_params[0][g];
            vpw[i] = new_params[1][g];
            const char *const from = reinterpret_cast<const char *>(new_codes[1]) + col * (CH / 2);
            if constexpr (CH < 8) vw[i][0] = *reinterpret_cast<const unsigned short *>(from);
            else words(from, vw[i]);
          }
      }
    }
    f32x4 sum[2];
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (j == 0) sum[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        const half8 kf = code_slots(kw[i][j], slots);
        sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[j], sum[i], 0, 0, 0);
        sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[j], sum[i], 0, 0, 0);
      }
    float s[8], top = NEG_INF;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = fmaf(half_lo(kpw[i]), fmaf(sum[i >> 2][i & 3], 512.0f, qsum8), half_hi(kpw[i]) * qsum);
      s[i] = groups_sum<NQ>(y);
    }
    if (more) load_k(c + kQ4Step);
    if (c + 32 > k1) {  // (rows past the range may hold anything)
      int left = k1 - c - 4 * t;
      asm volatile("" : "+v"(left));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key_of(i) >= left) {
          s[i] = NEG_INF;
          vpw[i] = 0;
        }
    }
    if constexpr (FEW) {
      if (c + 32 > all_end || c < all_begin) {
        int end = row_end - c - 4 * t, begin = row_begin - c - 4 * t;
        asm volatile("" : "+v"(end), "+v"(begin));
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = key_of(i) >= end || key_of(i) < begin ? NEG_INF : s[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i]);
    top = max32(max16(top));
    unsigned short step = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) step = max(step, (unsigned short)vpw[i]);  // (positive halves order as integers)
    if (__any(top > m || half_lo(step) > cap)) {
      const float mnew = fmaxf(m, top), largest = max32(max16(half_lo(step)));
      float alpha = fast_exp2((m - safe_max(mnew)) * inv);
      m = mnew;
      const bool far = fabsf(safe_max(m) * inv) >= 0x1p20f, was_far = cap > 0x1p100f;
      if (far ? !was_far : was_far || largest > cap) {
        // (steps are no less than 2^-24: past 2^40 the sums would only overflow)
        const unsigned to = far ? 127u << 23 : min(scale_to(largest, 14), 167u << 23);
        alpha *= __uint_as_float(to) * inverse_scale(scale);
        scale = to;
        cap = far ? __builtin_inff() : 60000.0f * inverse_scale(scale);
      }
      l *= alpha;
      omin *= alpha;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = __shfl(alpha, 4 * t + e);
#pragma unroll
        for (int n = 0; n < CH; ++n) o[n][e] *= f;
      }
    }
    const float shift = fmaf(-safe_max(m), inv, (float)((int)(scale >> 23) - 127));
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = fast_exp2(fmaf(s[i], inv, shift));
      l += w;
      p[i] = w * half_lo(vpw[i]);
      omin = fmaf(w, fmaf(half_lo(vpw[i]), 8.0f, half_hi(vpw[i])), omin);
    }
    half8 ph, pl;
    split8(p, minus_one, &ph, &pl);
#pragma unroll
    for (int n = 0; n < CH; ++n) {
      const half8 vf = value_slots<CH>(vw, n, slots);
      o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, vf, o[n], 0, 0, 0);
      o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, vf, o[n], 0, 0, 0);
    }
    if (more) load_v(c + kQ4Step);
  }

  if constexpr (STEP) {
    if (k1 == hi && hb == 0) {
      const long row = (long)h * seq_rows.cap + hi - 1;
      const int i = threadIdx.x;
      if (i < D / 4) {
        const int which = i / (D / 8), w = i % (D / 8);
        reinterpret_cast<unsigned *>((which ? seq_rows.v : seq_rows.k) + row * (D / 2))[w] =
            reinterpret_cast<const unsigned *>(new_codes[which])[w];
      } else if (i < D / 4 + 2 * G) {
        const int which = (i - D / 4) / G, w = (i - D / 4) % G;
        (which ? seq_rows.vp : seq_rows.kp)[row * G + w] = new_params[which][w];
      }
    }
  }

  l = sum32(sum16(l));
  omin = sum32(sum16(omin));
  const float unscale = inverse_scale(scale);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int row = 4 * t + e;
    const float least = __shfl(omin, row), back = __shfl(unscale, row);
    if (row / NQ == g)
#pragma unroll
      for (int n = 0; n < CH; ++n) red_o[wave][row % NQ][col * CH + n] = fmaf(o[n][e], 512.0f, least) * back;
  }
  if (lane < NQ) {
    red_l[wave][lane] = l * unscale;
    wave_m[wave][lane] = m == NEG_INF ? m : m * inv;
  }
  __syncthreads();
  const long entry = (((long)z * a.Hkv + h) * a.HB + hb) * a.max_splits + split;
#pragma unroll
  for (int e = threadIdx.x; e < NQ * D; e += 64 * kQ4Waves) {
    const int r = e / D, dim = e % D;
    if (hb * NQ + r >= rows) break;
    float M = NEG_INF;
#pragma unroll
    for (int w = 0; w < kQ4Waves; ++w) M = fmaxf(M, wave_m[w][r]);
    const float Ms = safe_max(M);
    float O = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kQ4Waves; ++w) {
      const float f = fast_exp2(wave_m[w][r] - Ms);
      O = fmaf(red_o[w][r][dim], f, O);
      L = fmaf(red_l[w][r], f, L);
    }
    if (a.max_splits > 1) {
      float *dst = a.partial + entry * (long)ENTRY;
      dst[e] = O;
      if (dim == 0) {
        dst[NQ * D + 2 * r] = M;
        dst[NQ * D + 2 * r + 1] = L;
      }
    } else {
      a.out[row_of(a, z, h, hb * NQ + r) * D + dim] = O / L;
      if (dim == 0 && !(L > 0.0f && L < __builtin_inff())) atomicOr(a.err, kDevErrSoftmaxDenominator);
    }
  }
}

// Merges the key ranges of one (query, KV head, head block): OUTS consecutive
// outputs x SL range lanes. The ranges' weights come first, a thread a range, so
// that the sums' reads depend on nothing and are all in flight at once.
template <int D, int MB, int OUTS, int SL>
__global__ __launch_bounds__(OUTS * SL) void q4_combine_kernel(const Q4AttnArgsOf<MB> a) {
  constexpr int NQ = 512 / D, ENTRY = NQ * (D + 2), WAVES = OUTS * SL / 64;
  __shared__ float weight[OUTS * SL], part[SL][OUTS + 1], wave_m[WAVES], wave_l[WAVES];
  const int z = blockIdx.z, hb = blockIdx.x % a.HB, h = blockIdx.x / a.HB;
  const int tid = threadIdx.x, e = blockIdx.y * OUTS + tid % OUTS, r = blockIdx.y * OUTS / D, sl = tid / OUTS;
  if (hb * NQ + r >= a.S * a.R) return;
  int lo, hi;
  visible(a, z, &lo, &hi);
  const int nsplit = (hi - lo + a.kps - 1) / a.kps;
  const float *ents = a.partial + (((long)z * a.Hkv + h) * a.HB + hb) * a.max_splits * (long)ENTRY;
  float em = NEG_INF, el = 0.0f;
  if (tid < nsplit) {
    const float2 ml = *reinterpret_cast<const float2 *>(ents + (long)tid * ENTRY + NQ * D + 2 * r);
    em = ml.x;
    el = ml.y;
  }
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = sl + i * SL;
    v[i] = s < nsplit ? ents[(long)s * ENTRY + e] : 0.0f;
  }
  const float top = max32(max16(row_max(em)));
  if ((tid & 63) == 0) wave_m[tid >> 6] = top;
  __syncthreads();
  const float M = safe_max(row_max(wave_m[tid % WAVES]));
  const float w = fast_exp2(em - M);
  if (tid < nsplit) weight[tid] = w;
  const float sum = group_sum<64>(tid < nsplit ? el * w : 0.0f);
  if ((tid & 63) == 0) wave_l[tid >> 6] = sum;
  __syncthreads();
  float O = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = sl + i * SL;
    if (s < nsplit) O = fmaf(v[i], weight[s], O);
  }
#pragma unroll 4
  for (int s = sl + 4 * SL; s < nsplit; s += SL) O = fmaf(ents[(long)s * ENTRY + e], weight[s], O);
  part[sl][tid % OUTS] = O;
  __syncthreads();
  if (tid < OUTS) {
    float total = 0.0f, L = 0.0f;
#pragma unroll
    for (int k = 0; k < SL; ++k) total += part[k][tid];
#pragma unroll
    for (int k = 0; k < WAVES; ++k) L += wave_l[k];
    a.out[row_of(a, z, h, hb * NQ + r) * D + e % D] = total / L;
    if ((e % D) == 0 && !(L > 0.0f && L < __builtin_inff())) atomicOr(a.err, kDevErrSoftmaxDenominator);
  }
}

namespace {

template <int D, int MB>
hipError_t attend(hipStream_t st, const Q4AttnArgsOf<MB> &a, int nz) {
  const dim3 grid((unsigned)(a.Hkv * a.HB), (unsigned)a.max_splits, (unsigned)nz);
  auto kernel = a.k ? q4_attend_kernel<D, MB, true, false> : q4_attend_kernel<D, MB, false, false>;
  if constexpr (MB == 1)
    if (a.S > 1) kernel = q4_attend_kernel<D, MB, false, true>;
  // One workgroup a CU where that is all there are: two, which heads of 64 have the
  // registers for, come together while other CUs stay empty, so LDS that nothing uses
  // keeps them apart. (16 sequences of 2432 to 8192 keys, 32 heads on 8 of 64: 28 us, 42
  // without. More workgroups go better two a CU: 16 of 1024 keys, 32 heads on 32, 16 us,
  // 19 with it.)
  long live = 0;
  for (int z = 0; z < nz; ++z) {
    const int keys = a.window > 0 ? (int)std::min<long>(a.seq[z].len, (long)a.window + a.S - 1) : a.seq[z].len;
    live += (keys + a.kps - 1) / a.kps * (long)grid.x;
  }
  const unsigned apart = D == 64 && live <= kQ4GridWorkgroups ? 62 * 1024 : 0;
  hipLaunchKernelGGL(kernel, grid, dim3(64 * kQ4Waves), apart, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.max_splits == 1) return e;
  // (32 range lanes for many ranges; two ranges of 16 sequences, 24 heads on 8 of 128:
  // 8.5 us with them, 3.3 with four)
  const unsigned outs = (unsigned)(std::min(a.S * a.R, 512 / D) * D), x = (unsigned)(a.Hkv * a.HB), z = (unsigned)nz;
  if (a.max_splits <= 16) hipLaunchKernelGGL((q4_combine_kernel<D, MB, 64, 4>), dim3(x, outs / 64, z), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((q4_combine_kernel<D, MB, 32, 32>), dim3(x, outs / 32, z), dim3(1024), 0, st, a);
  return hipGetLastError();
}

template <int D>
hipError_t attend_d(hipStream_t st, const Q4AttnArgs &a, int nz) {
  if (nz == 1) {
    Q4AttnArgsOf<1> one;
    static_cast<Q4AttnBase &>(one) = a;
    one.seq[0] = a.seq[0];
    return attend<D, 1>(st, one, nz);
  }
  return attend<D, kMaxDecodeBatch>(st, a, nz);
}

}  // namespace

bool q4_supported(size_t D) { return D == 64 || D == 128 || D == 256; }

Q4AttnPlan q4_attend_plan(int D, int rows, int Hkv, const int *keys, int n) {
  Q4AttnPlan p;
  p.RB = 512 / D;  // the kernel's rows
  p.HB = (rows + p.RB - 1) / p.RB;
  constexpr int chunk = kQ4Step;
  long total = 0;
  int most = 1;
  for (int i = 0; i < n; ++i) {
    total += keys[i];
    most = std::max(most, keys[i]);
  }
  const long heads = (long)Hkv * p.HB;
  const long per = (total * heads + kQ4GridWorkgroups - 1) / kQ4GridWorkgroups;
  long kps = std::max<long>(1, (per + chunk - 1) / chunk) * chunk;
  // Ragged lengths leave short last ranges: no more workgroups than are aimed at (or
  // one a head and sequence), which would wait for another to end. (16 sequences of
  // 2432 to 8192 keys, 24 heads on 8 of 128: 36 us, 46 without.)
  const long limit = std::max<long>(kQ4GridWorkgroups, n * heads);
  for (;;) {
    long wgs = 0;
    for (int i = 0; i < n; ++i) wgs += (keys[i] + kps - 1) / kps * heads;
    if (wgs <= limit) break;
    kps += std::max<long>(1, kps / chunk / 16) * chunk;
  }
  // Ranges cost a second launch, a step 1 to 2 us: short contexts stay one range.
  // (768 keys, heads of 64 7.2 us in one range, 7.2 in three, with one launch more for
  // the host; of 128 9.0 and 8.6; of 256 13.2 and 11.2, 512 keys 10.5 and 11.2.)
  const long one = (D == 256 ? 2 : 3) * chunk;
  if (most <= one) kps = one;
  if ((most + kps - 1) / kps > kMaxDecodeSplits)
    kps = ((most + kMaxDecodeSplits - 1) / kMaxDecodeSplits + chunk - 1) / chunk * chunk;
  p.kps = (int)kps;
  p.splits = (int)((most + kps - 1) / kps);
  long wgs = 0;
  for (int i = 0; i < n; ++i) wgs += (keys[i] + kps - 1) / kps * heads;
  const long steps = (wgs + kQ4GridWorkgroups - 1) / kQ4GridWorkgroups * ((std::min<long>(kps, most) + chunk - 1) / chunk);
  p.time = (D == 64 ? 3.5 + 1.6 * steps : D == 128 ? 4.0 + 2.1 * steps : 5.0 + 3.0 * steps) + (p.splits > 1 ? 3.0 : 0.0);
  return p;
}

hipError_t launch_q4_attend(hipStream_t st, const Q4AttnArgs &a, int D, int nz) {
  switch (D) {
    case 64: return attend_d<64>(st, a, nz);
    case 128: return attend_d<128>(st, a, nz);
    case 256: return attend_d<256>(st, a, nz);
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
  const size_t most = std::max<size_t>(1, kQ4LaunchThreads / (Hkv * (D / 8)));  // rows of a launch
  for (size_t at = 0; at < n; at += most) {
    const size_t rows = std::min(most, n - at), out = at * Hkv * D;
    Q4Rows from = s;
    from.first += (int)at;
    const dim3 grid((unsigned)((rows * Hkv * (D / 8) + 255) / 256), 2);
    hipLaunchKernelGGL(q4_rows_kernel, grid, dim3(256), 0, st, from, (int)rows, (int)Hkv, (int)D, k_out ? k_out + out : nullptr,
                       v_out ? v_out + out : nullptr);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace spissa
