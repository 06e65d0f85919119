// q4_chunk.hip -- attention of several queries over a KV cache held in 4 bits
// (q4_cache.hip has the format), on v_mfma_f32_16x16x32_f16 with f32 sums.
//
// The products are f32's in all but name. Scores: a code is a whole number and
// so exact in binary16; the queries, scaled by a power of two that takes their
// row's largest to 2^9..2^10, are two nearest binary16 pieces. A 32-channel
// group is the depth of one instruction, so its product is scaled by the key's
// step in f32, and the minima times the queries' group sums (three pieces) are
// one more instruction over the groups:
//   s = 2^-e (sum_g step_g (code . q)_g + sum_g min_g (sum q)_g).
// Output: the values, step * code + min scaled by a power of two that takes the
// largest of the workgroup's keys to 2^13..2^14, and the probabilities, times 2^14,
// are two pieces each, of whose four products the three above 2^-22 are taken.
//
// A workgroup takes 128 or 256 rows of a KV head, a row being a (query,
// query head of the group) pair with the head fastest, so that short chunks
// fill the instruction's 16 columns with heads. Per tile of keys it widens the
// codes into LDS once for all of them: the keys as they are, in the order in
// which lanes take the A operand, the values as two pieces of V^T. The scores
// are formed as S^T = K Q^T, so a lane has one row (column lane % 16) and four
// keys of each 16, and two such blocks are the B operand of O^T += V^T P^T
// without an exchange, the values' keys being stored in that order.
//
// Bound: the matrix cores beside the vector work of scaling, softmax, pieces and
// widening: of a SIMD's time at 512 queries over 8192 keys (24 heads on 8 of 128,
// 150 us with the merge, 330 TFLOP/s of the plain products) matrix instructions
// take half, and vector ones' issue, in which a matrix instruction takes two
// slots, three fifths; the two overlap in part.
#include <algorithm>
#include <type_traits>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

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

// Eight waves. A tile of 8192 / D keys is in LDS twice (this one and the next),
// as it came and widened. Between two barriers a wave widens its part of the next
// tile and computes its rows' part of this one, the first four waves in that
// order and the last four in the other: a SIMD has one of each, so the
// conversions of one run beside the matrix instructions of the other (one loop
// body, in which the two kinds have the barrier at different places). Within a
// wave the LDS reads run one step ahead of the instructions that need them.
template <int D, int NW>
__global__ __launch_bounds__(NW * 64, NW / 4) void q4_chunk_kernel(const Q4ChunkArgs a) {
  constexpr int BN = 8192 / D, G = D / 32, DT = D / 16, VB = BN / 32;
  constexpr int AH = NW == 16 ? 1 : 2;  // fragments of a step in registers, or of this one and the next
  constexpr int CB = BN * D / 2, PB = BN * G * 4, RAW = 2 * (CB + PB);  // bytes of a tile's codes and params
  static_assert(CB == 4096 && PB == 1024, "a tile has the same bytes for every D");
  __shared__ __attribute__((aligned(16))) half8 k_lds[2][BN * G * 4];
  __shared__ __attribute__((aligned(16))) half8 v_lds[2][2][VB * DT * 64];
  // (sixteen waves have the steps in binary16, half the LDS reads, in mixed-precision FMAs; eight in f32)
  typedef std::conditional_t<NW == 16, _Float16, float> step_t;
  typedef __attribute__((ext_vector_type(4))) step_t step4;
  __shared__ __attribute__((aligned(16))) step_t step_lds[2][BN * G];
  __shared__ __attribute__((aligned(16))) _Float16 min_lds[2][BN][8];
  __shared__ __attribute__((aligned(16))) char raw_lds[2][RAW];
  __shared__ __attribute__((aligned(16))) float most_lds[NW];

  float minus_one = -1.0f;
  unsigned base1024 = 0x64006400u;
  asm volatile("" : "+s"(minus_one));
  asm volatile("" : "+v"(base1024));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kq = lane >> 4;
  // Blocks of rows, the last (longest) ones of every head first; key ranges of each.
  // Ids equal modulo 8 share an XCD: where heads do not spread a block's ranges over
  // them, each range takes eight blocks in an order of its own. (2048 queries of 4 heads
  // on one of 256, six ranges: 70 us, 78 without; 32 heads on 8 of 64, two ranges, would
  // go from 85 to 94.)
  const int h = blockIdx.x, split = blockIdx.z;
  int order = blockIdx.y;
  if (a.Hkv % 8 != 0 && (order | 7) < (int)gridDim.y) order = (order & ~7) | ((order + split) & 7);
  const int block = gridDim.y - 1 - order;
  const int rows = a.S * a.R;
  const int row0 = block * (NW * 16) + wave * 16;
  const int P = a.len - a.S;  // the first query's position
  // keys that any row of the workgroup sees
  const int first_q = block * (NW * 16) / a.R, last_q = min(rows - 1, (block + 1) * (NW * 16) - 1) / a.R;
  const int hi = a.causal ? P + last_q + 1 : a.len;
  const int lo = a.window > 0 ? max(0, P + first_q + 1 - a.window) : 0;
  const int t0 = lo / BN + split * a.tps;
  const int t1 = min((hi + BN - 1) / BN, t0 + a.tps);

  // A lane's row, for the column.
  const int pos = P + min(row0 + col, rows - 1) / a.R;
  const long orow = [&] {  // query * Hq + head
    const int r = min(row0 + col, rows - 1), query = r / a.R;
    return (long)query * a.Hq + h * a.R + (r - query * a.R);
  }();
  const long total = (long)a.S * a.Hq;
  float *const ml = a.part_ml + ((long)split * total + orow) * 2;
  if (t0 >= t1) {  // (a range of none of the block's tiles: with m at -inf no outputs are read)
    if (row0 + col < rows && kq == 0) *reinterpret_cast<float2 *>(ml) = make_float2(NEG_INF, 0.0f);
    return;
  }

  // A tile's codes, steps and minima come as they are, straight into LDS (1 KB a
  // wave and instruction). The rows past the last are read too (the buffers end
  // 128 rows later) and may hold anything: their keys are hidden, and their
  // values taken as zeros.
  const long head = (long)h * a.rows.cap;
  const char *src[4] = {reinterpret_cast<const char *>(a.rows.k) + head * (D / 2),
                        reinterpret_cast<const char *>(a.rows.v) + head * (D / 2),
                        reinterpret_cast<const char *>(a.rows.kp + head * G), reinterpret_cast<const char *>(a.rows.vp + head * G)};
  auto fetch = [&](int tile) {
#pragma unroll
    for (int i = 0; i < (RAW / 1024 + NW - 1) / NW; ++i) {
      const int chunk = i * NW + wave;  // keys' codes 4, values' codes 4, keys' params 1, values' params 1
      if (chunk >= RAW / 1024) continue;
      const int part = chunk < 4 ? 0 : chunk < 8 ? 1 : chunk - 6;
      const char *from = (part == 0 ? src[0] : part == 1 ? src[1] : part == 2 ? src[2] : src[3]) +
                         (long)tile * (part < 2 ? CB : PB) + (part < 2 ? (chunk & 3) * 1024 : 0);
      copy16(from, lane * 16, raw_lds[tile & 1] + chunk * 1024);
    }
  };
  fetch(t0);
  if (t0 + 1 < t1) fetch(t0 + 1);
  // The largest value of the range's rows, which their steps and minima bound, beside
  // the first tiles on their way: 0 to 2 % of the time. (A bound kept with the cache
  // would outlive rows that are taken back, and one of each tile takes 3 to 8 %.)
  {
    constexpr int AT_ONCE = 4;  // loads of a lane in flight
    typedef u32x4 __attribute__((aligned(4))) params_t;
    const params_t *const params = reinterpret_cast<const params_t *>(src[3] + (long)t0 * PB);
    const int words = (min(t1 * BN, a.len) - t0 * BN) * G, vectors = (words + 3) / 4;
    float most = 0.0f;
    for (int i = tid; i < vectors; i += NW * 64 * AT_ONCE) {
      u32x4 p[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) p[u] = params[min(i + u * NW * 64, vectors - 1)];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        if (G == 2 && 4 * min(i + u * NW * 64, vectors - 1) + 2 == words) p[u].z = p[u].w = 0;  // (an odd last row)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          most = fmaxf(most, fmaxf(fabsf(half_hi(p[u][j])), fabsf(fmaf(half_lo(p[u][j]), 15.0f, half_hi(p[u][j])))));
      }
    }
    most = wave_max(most);
    if (lane == 0) most_lds[wave] = most;
  }

  half8 qh[G], ql[G], qs;
  float inv;
  const float *q = a.q + orow * D + 8 * kq;
  float v[G][8], most = 0.0f;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float4 x = *reinterpret_cast<const float4 *>(q + 32 * g), y = *reinterpret_cast<const float4 *>(q + 32 * g + 4);
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
  inv = inverse_scale(sb);
  const float scale = __uint_as_float(sb);
  float sums[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[g][i] *= scale;
      sums[g] += v[g][i];
    }
    split8(v[g], minus_one, &qh[g], &ql[g]);
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
  qs = kq == 0 ? s0 : kq == 1 ? s1 : kq == 2 ? s2 : none;
  int wave_hi = 0, wave_lo = 0x7fffffff;  // keys that any row of the wave sees
  const int r = row0;
  if (r < rows) {
    wave_hi = max(wave_hi, a.causal ? P + min(rows - 1, r + 15) / a.R + 1 : a.len);
    wave_lo = min(wave_lo, a.window > 0 ? max(0, P + r / a.R + 1 - a.window) : 0);
  }

  f32x4 o[DT];
  float m, l;
  m = NEG_INF;
  l = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  unsigned vsb;  // the values' scale, as float bits
  float vscale;

  // A thread's share of a tile: half a key's group of 32 channels, and eight keys
  // (4 q + 0..3 and 16 + 4 q + 0..3 of 32) of two channels of the values.
  // (sixteen waves: the first eight have the values, the last eight the keys)
  const int part = tid & 511;
  const int kkey = (part & 15) + 16 * (part / (32 * G)), kg = (part >> 4) % G, khalf = part / (16 * G) & 1;
  const int vd = part % (D / 2) * 2, vq = part / (D / 2) % 4, vb = part / (2 * D);
  auto widen_k = [&](int tile) {
    const int buf = tile & 1;
    const char *const raw = raw_lds[buf];
    const uint2 kw = *reinterpret_cast<const uint2 *>(raw + (kkey * G + kg) * 16 + khalf * 8);
    const unsigned kp = *reinterpret_cast<const unsigned *>(raw + 2 * CB + (kkey * G + kg) * 4);
    half8 *const dst = &k_lds[buf][((kkey >> 4) * G + kg) * 64 + khalf * 32 + (kkey & 15)];
    dst[0] = codes8h(kw.x, base1024);
    dst[16] = codes8h(kw.y, base1024);
    if (khalf == 0) {
      step_lds[buf][((kkey >> 4) * G + kg) * 16 + (kkey & 15)] = (step_t)__builtin_bit_cast(_Float16, (unsigned short)kp);
      min_lds[buf][kkey][kg] = __builtin_bit_cast(_Float16, (unsigned short)(kp >> 16));
    }
  };
  auto widen_v = [&](int tile) {
    const int buf = tile & 1;
    const char *const raw = raw_lds[buf];
    const char *const params = raw + 2 * CB + PB + ((32 * vb + 4 * vq) * G + vd / 32) * 4;
    const unsigned char *const codes = reinterpret_cast<const unsigned char *>(raw) + CB + (32 * vb + 4 * vq) * (D / 2) + vd / 2;
    unsigned vw[8];
    float st[8], mn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned p = *reinterpret_cast<const unsigned *>(params + ((i & 3) + 16 * (i >> 2)) * (G * 4));
      vw[i] = codes[((i & 3) + 16 * (i >> 2)) * (D / 2)];
      st[i] = fmaf(half_lo(p), vscale, 0.0f);  // (one mixed-precision instruction)
      mn[i] = fmaf(half_hi(p), vscale, 0.0f);
    }
    if ((tile + 1) * BN > a.len) {
      int left = a.len - tile * BN - 32 * vb - 4 * vq;
      asm volatile("" : "+v"(left));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((i & 3) + 16 * (i >> 2) >= left) st[i] = mn[i] = 0.0f;
    }
    const int dt = vd >> 4;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(st[i], (float)(j ? vw[i] >> 4 : vw[i] & 15u), mn[i]);
      half8 vh, vl;
      split8(v, minus_one, &vh, &vl);
      // (the low bits mixed with the channel tile: the writes of a wave fall on all banks)
      const int at = (vb * DT + dt) * 64 + ((vq * 16 + (vd & 15) + j) ^ (dt & 7));
      v_lds[buf][0][at] = vh;
      v_lds[buf][1][at] = vl;
    }
  };
  auto widen = [&](int tile) {
    if (NW == 8 || wave >= 8) widen_k(tile);
    if (NW == 8 || wave < 8) widen_v(tile);
  };

  auto compute = [&](int tile) {
    const int buf = tile & 1, base = tile * BN;
    if (base >= wave_hi || base + BN <= wave_lo) return;
    // 32 keys at a time: their scores, the rows' maximum, the weights, the output.
    // (The earlier a wave is in its 32 keys, the more it goes before the others of its
    // SIMD, so that they come apart: 512 queries over 8192 keys, 24 heads on 8 of 128
    // 148 us against 155, a prompt of 2048 of 32 heads on 8 of 64 87 against 100.)
#pragma unroll 1
    for (int b = 0; b < VB; ++b) {
      const int key0 = base + 32 * b;
      if (key0 >= wave_hi || key0 + 32 <= wave_lo) continue;
      // Steps of two groups of one 16 keys; those instructions that depend on
      // each other are two apart.
      constexpr int NS = G;
      half8 kf[AH][2], mf[2];
      step4 st[AH][2];
      f32x4 s[2];
      const half8 *const kl = &k_lds[buf][2 * b * G * 64 + lane];
      const step_t *const sl = &step_lds[buf][2 * b * G * 16 + 4 * kq];
      auto load_k = [&](int step) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kf[step % AH][i] = kl[(2 * step + i) * 64];
          st[step % AH][i] = *reinterpret_cast<const step4 *>(sl + (2 * step + i) * 16);
        }
      };
      half8 vh[AH][2], vl[AH][2];
      // (one address a tile, its low bits mixed anew for each read)
      unsigned v_at = buf * (unsigned)sizeof v_lds[0] + b * (DT * 1024) + lane * 16;
      asm volatile("" : "+v"(v_at));
      auto load_v = [&](int step) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = 2 * step + i;
          const char *const at = reinterpret_cast<const char *>(v_lds) + (v_at ^ ((d & 7) * 16)) + d * 1024;
          vh[step % AH][i] = *reinterpret_cast<const half8 *>(at);
          vl[step % AH][i] = *reinterpret_cast<const half8 *>(at + sizeof v_lds[0][0]);
        }
      };
      mf[0] = *reinterpret_cast<const half8 *>(min_lds[buf][32 * b + col]);
      mf[1] = *reinterpret_cast<const half8 *>(min_lds[buf][32 * b + 16 + col]);
      if (AH == 2) load_k(0);
      __builtin_amdgcn_s_setprio(2);
#pragma unroll
      for (int step = 0; step < NS; ++step) {
        const int k = step / (G / 2), g = 2 * step % G;
        if (AH == 1) load_k(step);
        else if (step + 1 < NS) load_k(step + 1);
        else load_v(0);
        f32x4 c[2];
        if (g == 0) {
          s[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(mf[k], qs, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[step % AH][i], ql[g + i], (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[step % AH][i], qh[g + i], c[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[k][e] = fmaf((float)st[step % AH][i][e], c[i][e], s[k][e]);
        // (the sums stay in their step: left to itself the compiler keeps every step's products until the last)
        asm volatile("" : "+v"(s[k]));
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(1);
      half8 ph, pl;
      // (32 keys that every row sees need no mask: uniform over the wave)
      const int r = row0;
      const bool whole = r + 15 < rows && key0 + 32 <= (a.causal ? P + r / a.R + 1 : a.len) &&
                         key0 >= (a.window > 0 ? P + (r + 15) / a.R + 1 - a.window : 0);
      if (!whole) {
        const int kend = r + col < rows ? (a.causal ? pos + 1 : a.len) : 0;
        const int kbeg = a.window > 0 ? pos + 1 - a.window : 0;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * k + 4 * kq + e;
            if (key >= kend || key < kbeg) s[k][e] = NEG_INF;
          }
      }
      float top = NEG_INF;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[k][e]);
      top = max32(max16(top)) * inv;
      // A weight is exp2(score - m), and m is set 14 below the largest score, which has
      // the weight 2^14, and rises when a score passes it by 15.9: weights stay in
      // binary16's range, and the second piece, which ends at 2^-24, leaves two whole
      // pieces down to 2^-16 of the largest. (Keys of little weight count where the key
      // that has most of it has no value. 12 and 15.9, which scale the output anew less
      // often, take 1 % off 2048 queries.) Scores past 2^20, whose digits 14 would be
      // lost in, are references themselves.
      if (__any(top - m > 15.9f)) {
        const float mnew = fmaxf(m, fabsf(top) < 0x1p20f ? top - 14.0f : top);
        const float alpha = fast_exp2(m - safe_max(mnew));
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] *= alpha;
      }
      const float shift = -safe_max(m);
      float p[8];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * k + e] = fast_exp2(fmaf(s[k][e], inv, shift));
          l += p[4 * k + e];
        }
      split8(p, minus_one, &ph, &pl);
      __builtin_amdgcn_sched_barrier(0);
      // steps of two channel tiles
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int step = 0; step < DT / 2; ++step) {
        if (AH == 1) load_v(step);
        else if (step + 1 < DT / 2) load_v(step + 1);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          o[2 * step + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[step % AH][i], ph, o[2 * step + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          o[2 * step + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[step % AH][i], pl, o[2 * step + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          o[2 * step + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[step % AH][i], ph, o[2 * step + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  if constexpr (G < 8) {
    for (int i = tid; i < 2 * BN; i += NW * 64)
#pragma unroll
      for (int g = G; g < 8; ++g) min_lds[i & 1][i >> 1][g] = (_Float16)0.0f;
  }
  // Barrier i: tile i is widened, tile i + 1 has come, and tile i - 1 is no longer
  // read. The first waves widen tile i + 1 after it, the last ones before barrier
  // i + 1, after computing tile i.
  const bool ahead = (wave & 4) == 0;
  auto barrier = [&](int tile) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (tile + 2 < t1) fetch(tile + 2);
  };
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the first two tiles have come
  float largest = 0.0f;
#pragma unroll
  for (int i = 0; i < NW; ++i) largest = fmaxf(largest, most_lds[i]);
  vsb = __builtin_amdgcn_readfirstlane(scale_to(largest, 13));
  vscale = __uint_as_float(vsb);
#pragma unroll 1
  for (int tile = t0 - 1; tile < t1; ++tile) {
    if (ahead && tile >= t0) barrier(tile);
    const int next = ahead ? tile + 1 : tile;
    if (next >= t0 && next < t1) widen(next);
    if (!ahead && tile >= t0) barrier(tile);
    if (tile >= t0) compute(tile);
  }

  const float vinv = inverse_scale(vsb);
  const float sum = sum32(sum16(l));
  if (row0 + col >= rows) return;
  float *dst;
  float f;
  if (a.splits > 1) {
    if (kq == 0) *reinterpret_cast<float2 *>(ml) = make_float2(m, sum);
    if (m == NEG_INF) return;
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
        make_float4(o[d][0] * f, o[d][1] * f, o[d][2] * f, o[d][3] * f);
}

namespace {

template <int D, int NW>
hipError_t chunk(hipStream_t st, const Q4ChunkArgs &a) {
  const long rows = (long)a.S * a.R;
  const dim3 grid((unsigned)a.Hkv, (unsigned)((rows + NW * 16 - 1) / (NW * 16)), (unsigned)a.splits);
  hipLaunchKernelGGL((q4_chunk_kernel<D, NW>), grid, dim3(NW * 64), 0, st, a);
  return hipGetLastError();
}

}  // namespace

// The rows of a workgroup and the ranges of its keys that a model of the launch
// finds fastest: a workgroup takes 3 us and a time for each tile, the CUs take the
// workgroups longest first, and ranges are merged at 2.2 MB a us after 3.5 us.
// Measured and modelled, us: a prompt of 2048, 24 heads on 8 of 128, in blocks of
// 256 rows with two ranges 101 and 102, with one 140 and 147, of 128 rows with one
// 106 and 104; 512 queries over 8192 keys, 256 rows with five ranges 147 and 135,
// four 158 and 162, 16 174 and 165; 2048, 4 heads on 2 of 256, three ranges 81 and
// 88, one 164 and 165.
Q4ChunkPlan q4_chunk_plan(int D, int S, int R, int Hkv, int len, int causal, int window, int cus) {
  const int BN = 8192 / D;
  const long rows = (long)S * R;
  Q4ChunkPlan best;
  for (int per = 128; per <= (D < 256 && rows > 128 ? 256 : 128); per += 128) {
    const double tile = D == 256 ? 2.45 : D == 128 ? (per == 256 ? 4.2 : 3.0) : per == 256 ? 5.2 : 3.9;
    const long blocks = (rows + per - 1) / per;
    auto tiles_of = [&](long block) {  // as the kernel has them
      const long first = block * per / R, last = std::min(rows - 1, (block + 1) * per - 1) / R;
      const long hi = causal ? len - S + last + 1 : len, lo = window > 0 ? std::max<long>(0, len - S + first + 1 - window) : 0;
      return (hi + BN - 1) / BN - lo / BN;
    };
    long most = 1;
    for (long b = 0; b < blocks; ++b) most = std::max(most, tiles_of(b));
    int last_splits = 0;
    for (long want = 1; want <= 64 && (want == 1 || want * blocks * Hkv <= 4L * cus); ++want) {
      const long tps = (most + want - 1) / want;
      const int splits = (int)((most + tps - 1) / tps);
      if (splits == last_splits) continue;
      last_splits = splits;
      double sum = 0.0, least = 1e30;
      long pieces = 0;
      for (long b = 0; b < blocks; ++b) {
        const long n = tiles_of(b), k = (n + tps - 1) / tps;
        pieces += k;
        sum += n * tile + 3.0 * k;
        least = std::min(least, (n - (k - 1) * tps) * tile + 3.0);
      }
      const long n = pieces * Hkv, full = n / cus * cus;
      const double longest = tps * tile + 3.0;
      // (CUs that get one workgroup more than the others: by how much at least)
      double time = std::max(longest, sum * Hkv / cus + (n > cus && n > full ? least * (1.0 - (double)(n - full) / cus) : 0.0));
      if (splits > 1) time += 3.5 + (double)splits * rows * Hkv * D * sizeof(float) / 2.2e6;
      if (best.time == 0.0 || time < best.time) {
        best.time = time;
        best.per = per;
        best.splits = splits;
        best.tps = (int)tps;
      }
    }
  }
  best.time += 3.0;  // (the launch)
  if (best.splits > 1) best.partial_bytes = (size_t)best.splits * rows * Hkv * (D + 2) * sizeof(float);
  return best;
}

hipError_t launch_q4_chunk(hipStream_t st, const Q4ChunkArgs &a, int D) {
  const bool wide = a.per == 256;
  switch (D) {
    case 64: return wide ? chunk<64, 16>(st, a) : chunk<64, 8>(st, a);
    case 128: return wide ? chunk<128, 16>(st, a) : chunk<128, 8>(st, a);
    case 256: return chunk<256, 8>(st, a);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace spissa
