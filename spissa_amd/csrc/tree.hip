// tree.hip -- decoding with drafted tokens: a tree of them through one layer's
// attention, the walk along those that sampling confirms, and the move of their
// rows in the caches.
//
// The step. Node t of a sequence of P cached rows has the position P + depth(t)
// and sees the cached rows (with a window those less than W positions before it),
// the nodes it descends from and itself. Its key, rotated at its position, and its
// value become the cache's row P + t, and
//   out_t = sum_j p_tj v_j,  p_t = softmax_j(q_t . k_j / sqrt(d)).
#include <algorithm>
#include <type_traits>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

constexpr int kMaskWords = kTreeMaxNodes / 32;

// The nodes' depths and the nodes that each sees (with a window those less than it
// apart), by doubling: after k rounds a node knows the 2^k nodes above it. A parent out
// of its range counts as none.
struct TreeShape {
  int depth[kTreeMaxNodes];
  int above[kTreeMaxNodes];  // the node 2^k above
  unsigned mask[kTreeMaxNodes][kMaskWords];
};
// What is further than the window above node t is not seen.
__device__ __forceinline__ void narrow(int t, int window, TreeShape &s) {
  const int depth = s.depth[t];
  if (window > 0 && depth >= window)
    for (int j = 0; j < t; ++j)
      if (depth - s.depth[j] >= window) s.mask[t][j >> 5] &= ~(1u << (j & 31));
}
// Up to 64 nodes: by one wave, without a barrier. p: the lane's node's parent.
__device__ __forceinline__ void shape_of_wave(int p, int nodes, int window, TreeShape &s, int *err) {
  const int t = threadIdx.x & 63;
  if (p < -1 || p >= t) {
    if (err && t < nodes) atomicOr(err, kDevErrTreeParent);
    p = -1;
  }
  int depth = p >= 0 ? 1 : 0;
  unsigned lo = t < 32 ? 1u << t : 0u, hi = t < 32 ? 0u : 1u << (t - 32);
  while (__any(p >= 0)) {
    const int from = p < 0 ? t : p;
    const int d = __shfl(depth, from), up = __shfl(p, from);
    const unsigned l = (unsigned)__shfl((int)lo, from), h = (unsigned)__shfl((int)hi, from);
    if (p >= 0) {
      depth += d;
      lo |= l;
      hi |= h;
      p = up;
    }
  }
  s.depth[t] = depth;
  s.mask[t][0] = lo;
  s.mask[t][1] = hi;
  if (window > 0 && t < nodes) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    narrow(t, window, s);
  }
}
// More nodes: two threads a node, each with half of its words.
__device__ __forceinline__ void shape_of_workgroup(int p, int nodes, int window, TreeShape &s, int *err) {
  constexpr int HALF = kMaskWords / 2;
  const int t = threadIdx.x & (kTreeMaxNodes - 1), w0 = threadIdx.x / kTreeMaxNodes * HALF;
  if (p < -1 || p >= t) {
    if (err && t < nodes) atomicOr(err, kDevErrTreeParent);
    p = -1;
  }
  int depth = p >= 0 ? 1 : 0;
  unsigned m[HALF];
#pragma unroll
  for (int w = 0; w < HALF; ++w) m[w] = t >> 5 == w0 + w ? 1u << (t & 31) : 0u;
  for (;;) {
    if (w0 == 0) {
      s.depth[t] = depth;
      s.above[t] = p;
    }
#pragma unroll
    for (int w = 0; w < HALF; ++w) s.mask[t][w0 + w] = m[w];
    if (!__syncthreads_or(p >= 0)) break;
    if (p >= 0) {
      depth += s.depth[p];
#pragma unroll
      for (int w = 0; w < HALF; ++w) m[w] |= s.mask[p][w0 + w];
      p = s.above[p];
    }
    __syncthreads();
  }
  if (window > 0) {
    if (w0 == 0 && t < nodes) narrow(t, window, s);
    __syncthreads();
  }
}

__device__ __forceinline__ unsigned wave_max_bits(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xf, 0xf, false));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xf, 0xf, false));
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}
__device__ __forceinline__ float unbits(unsigned b) { return __uint_as_float(b); }

// Channels 4 l..4 l + 3 and their rotation's partners, half a row on, of row `row`.
template <int D>
__device__ __forceinline__ void load_pairs(const float *row, int l, f32x4 &lo, f32x4 &hi) {
  lo = *reinterpret_cast<const f32x4 *>(row + 4 * l);
  hi = *reinterpret_cast<const f32x4 *>(row + D / 2 + 4 * l);
}
// The norm's weights times 1 / rms on such channels.
template <int D>
__device__ __forceinline__ void norm_pairs(f32x4 &lo, f32x4 &hi, const float *w, int l, float inv) {
#pragma clang fp contract(off)
  f32x4 a, b;
  load_pairs<D>(w, l, a, b);
  lo = lo * inv * a;
  hi = hi * inv * b;
}
__device__ __forceinline__ void rotate_pairs(f32x4 &lo, f32x4 &hi, const float *cos, const float *sin, long at) {
  const f32x4 c = *reinterpret_cast<const f32x4 *>(cos + at), s = *reinterpret_cast<const f32x4 *>(sin + at);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = lo[i], y = hi[i];
    rotate_pair(x, y, c[i], s[i]);
    lo[i] = x;
    hi[i] = y;
  }
}
__device__ __forceinline__ float squares(const f32x4 &a, const f32x4 &b) {
#pragma clang fp contract(off)
  return ((a[0] * a[0] + b[0] * b[0]) + (a[1] * a[1] + b[1] * b[1])) + ((a[2] * a[2] + b[2] * b[2]) + (a[3] * a[3] + b[3] * b[3]));
}

}  // namespace

// Eight waves. A row is a node and one of the KV head's query heads; a wave has NB
// blocks of 16 rows and, of each tile of 8192 / D keys, all (heads of 256) or half
// (waves 0..3 the first, 4..7 the second; the halves meet at the end). Tiles are first
// the cached rows from the first that any node sees, then the nodes' own. A tile comes
// into registers while the one before is computed; waves 0..3 take its values, waves
// 4..7 its keys, and write them to LDS once for all rows as two binary16 pieces, in
// the order in which lanes take the operands. S^T = K Q^T, so a lane has one row
// (column lane % 16) and four keys of each 16, and two such blocks are the B operand
// of O^T += V^T P^T without an exchange, the values' keys being stored in that order.
// Channels of the scores' product come as 4 l..4 l + 3 beside D / 2 + 4 l..., which
// makes a rotation's pairs neighbours in a lane.
//
// Scales. Pieces hold 2^-23 of a number only between 2^-3 and 2^16. Keys and values
// are multiplied by a power of two that takes the first tile's largest to 2^11..2^12.
// Each tile's largest is known after it is written; one that does not fit (or is not
// finite) is loaded and written again, with the scale that it needs, the output so
// far following, or, where a number is not finite, with zeros in its place and its key
// noted: rows that see such a key become NaN.
//
// Grid: (KV heads, splits, sequences x blocks of rows).
template <int D, int KW, int MB>
__global__ __launch_bounds__(512, 2) void tree_attend_kernel(const TreeArgsOf<MB> a) {
  constexpr int BN = 8192 / D, G = D / 32, DT = D / 16, VB = BN / 32, KB = BN / 16, TR = D / 8;
  constexpr int NB = 1, RW = 8 / KW, ROWS = RW * NB * 16;
  constexpr int KBW = KB / KW, VBW = VB / KW;  // a wave's 16 and 32 keys of a tile
  static_assert(KB * G == 16 && VB * DT == 16, "a tile has 8192 keys' and as many values' channels");
  __shared__ __attribute__((aligned(16))) half8 pieces_lds[2][2][2][1024];  // values, buffer, piece
  half8 (*const kp_lds)[2][1024] = pieces_lds[0], (*const vp_lds)[2][1024] = pieces_lds[1];
  __shared__ TreeShape shape;
  __shared__ unsigned most_lds[2][8];
  __shared__ unsigned bad_lds[VB];

  float minus_one = -1.0f;
  asm volatile("" : "+s"(minus_one));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int col = lane & 15, kq = lane >> 4;
  const int rw = wave % RW, kw = wave / RW;
  const int h = blockIdx.x, split = blockIdx.y, b = blockIdx.z / a.blocks, block = blockIdx.z - b * a.blocks;
  const int past = a.seq[b].past, nodes = a.seq[b].nodes, seq_first = a.seq[b].first;
  const int rows = nodes * a.R;
  if (block * ROWS >= rows) return;
  const int lo = a.window > 0 ? max(0, past + 1 - a.window) : 0;
  const int cached = (past - lo + BN - 1) / BN, tiles = cached + (nodes + BN - 1) / BN;
  const int t0 = split * a.tps, t1 = min(tiles, t0 + a.tps);

  // Rows of the wave: blocks rw, rw + RW, ... of 16.
  int node[NB];
  long orow[NB];
  bool live[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = block * ROWS + (n * RW + rw) * 16 + col, r = min(row, rows - 1);
    live[n] = row < rows;
    node[n] = r / a.R;
    orow[n] = (long)(seq_first + node[n]) * a.Hq + h * a.R + (r - node[n] * a.R);
  }
  auto busy = [&](int n) __attribute__((always_inline)) { return block * ROWS + (n * RW + rw) * 16 < rows; };
  auto part = [&](int n) __attribute__((always_inline)) { return a.part + ((long)split * a.total + orow[n]) * (D + 4); };
  if (t0 >= t1) {  // (no keys: nothing of the row's part is read)
#pragma unroll
    for (int n = 0; n < NB; ++n)
      if (live[n] && kq == 0 && kw == 0) *reinterpret_cast<float2 *>(part(n) + D) = make_float2(NEG_INF, 0.0f);
    return;
  }

  // A thread's share of a tile: of values eight keys (4 q + 0..3 and 16 + 4 q + 0..3 of
  // 32) of four channels; of keys, four rows' channels 4 l.. and D / 2 + 4 l... Load i
  // has the key thread_key + step_key(i, values).
  const bool values = wave < 4;
  const int part_of = tid & 255;
  const int vg = part_of / (D / 4);
  int vl = part_of % (D / 4), vb0 = vg >> 2, vq = vg & 3;
  int kl = part_of % TR, kk = part_of / TR;
  int thread_key = values ? vb0 * 32 + 4 * vq : kk, thread_channel = values ? 4 * vl : 4 * kl;
  const long stride = (long)a.Hkv * D;
  float *const cache_rows = (values ? +a.seq[b].v : +a.seq[b].k) + h * D;
  const float *const own_rows = (values ? +a.v : +a.k) + seq_first * stride + h * D;
  f32x4 raw[8];
  auto step_key = [&](int i, auto values) __attribute__((always_inline)) { return values ? (i & 3) + 16 * (i >> 2) : (i >> 1) * (256 / TR); };
  auto load = [&](int tile, auto values) __attribute__((always_inline)) {
    const bool own = tile >= cached;
    const int first = own ? (tile - cached) * BN : lo + tile * BN, left = (own ? nodes : past) - first;
    const char *const src = reinterpret_cast<const char *>((own ? own_rows : +cache_rows) + first * stride);
    if (left >= BN) {
      const unsigned off = (unsigned)(thread_key * stride + thread_channel) * 4u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        raw[i] = *reinterpret_cast<const f32x4 *>(src + (step_key(i, values) * stride + (values ? 0 : (i & 1) * (D / 2))) * 4 + off);
    } else {  // (rows past the last: that one again)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long at = min(thread_key + step_key(i, values), left - 1) * stride + thread_channel + (values ? 0 : (i & 1) * (D / 2));
        raw[i] = *reinterpret_cast<const f32x4 *>(src + at * 4);
      }
    }
  };
  // The nodes' own rows: the norm and the rotation of keys, and the append.
  auto finish = [&](int tile, auto values, f32x4 (&cur)[8]) __attribute__((always_inline)) {
    const int first = (tile - cached) * BN + thread_key;
    if (!values) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int t = min(first + step_key(i, values), nodes - 1);
        if (a.k_norm) {
          const float inv = 1.0f / sqrtf(group_sum<TR>(squares(cur[i], cur[i + 1])) / (float)D + a.eps);
          norm_pairs<D>(cur[i], cur[i + 1], a.k_norm, kl, inv);
        }
        if (a.cos) rotate_pairs(cur[i], cur[i + 1], a.cos, a.sin, (long)(past + shape.depth[t]) * (D / 2) + 4 * kl);
      }
    }
    if (block != 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = first + step_key(i, values);
      if (t < nodes)
        *reinterpret_cast<f32x4 *>(cache_rows + (past + t) * stride + thread_channel + (values ? 0 : (i & 1) * (D / 2))) = cur[i];
    }
  };
  // The wave's largest magnitude, as bits (a NaN or an infinity is above the rest).
  auto post = [&](int slot, const f32x4 (&cur)[8]) __attribute__((always_inline)) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = max(m, max(__float_as_uint(cur[i][0]) & 0x7fffffffu, __float_as_uint(cur[i][1]) & 0x7fffffffu));
      m = max(m, max(__float_as_uint(cur[i][2]) & 0x7fffffffu, __float_as_uint(cur[i][3]) & 0x7fffffffu));
    }
    m = wave_max_bits(m);
    if (lane == 0) most_lds[slot][wave] = m;
  };
  unsigned kbits = 127u << 23, vbits = 127u << 23;  // the scales, as float bits
  auto write = [&](int buf, auto values, const f32x4 (&cur)[8]) __attribute__((always_inline)) {
    const float scale = unbits(values ? vbits : kbits);
    if (values) {
      const int dt = vl >> 2;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = cur[i][c] * scale;
        half8 ph, pl;
        split8(v, minus_one, &ph, &pl);
        // (the low bits mixed: the writes of a wave fall on all banks)
        const int at = (vb0 * DT + dt) * 64 + vq * 16 + ((4 * (vl & 3) + c) ^ (dt & 3));
        vp_lds[buf][0][at] = ph;
        vp_lds[buf][1][at] = pl;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float v[8] = {cur[i][0] * scale,     cur[i][1] * scale,     cur[i][2] * scale,     cur[i][3] * scale,
                            cur[i + 1][0] * scale, cur[i + 1][1] * scale, cur[i + 1][2] * scale, cur[i + 1][3] * scale};
        half8 ph, pl;
        split8(v, minus_one, &ph, &pl);
        const int key = thread_key + step_key(i, values), at = ((key >> 4) * G + (kl >> 2)) * 64 + (kl & 3) * 16 + ((key ^ kl) & 15);
        kp_lds[buf][0][at] = ph;
        kp_lds[buf][1][at] = pl;
      }
    }
  };
  auto largest = [&](int slot, int from) __attribute__((always_inline)) {
    const uint4 m = *reinterpret_cast<const uint4 *>(most_lds[slot] + from);
    return max(max(m.x, m.y), max(m.z, m.w));
  };

  // (all that needs no other load first: the parents, the queries, the first tile)
  const int own_node = tid & (nodes > 64 ? kTreeMaxNodes - 1 : 63), parent = own_node < nodes ? a.parents[seq_first + own_node] : -1;
  half8 qh[NB][G], ql[NB][G];
  float inv_q[NB];
  int row_lo[NB], wave_lo = 0;  // keys from row_lo on are seen by the row, from wave_lo on by all rows of the wave
  {
    f32x4 x[NB][G], y[NB][G];
#pragma unroll
    for (int n = 0; n < NB; ++n)
      if (busy(n)) {
#pragma unroll
        for (int g = 0; g < G; ++g) load_pairs<D>(a.q + orow[n] * D, 4 * g + kq, x[n][g], y[n][g]);
      }
    load(t0, values);
    int *const err = block == 0 && split == 0 && h == 0 ? a.err : nullptr;
    if (nodes > 64) {
      shape_of_workgroup(parent, nodes, a.window, shape, err);
    } else {
      // (a wave that is the last to have rows)
      if (wave == 7) shape_of_wave(parent, nodes, a.window, shape, err);
      __syncthreads();
    }
    // The queries, as the B operand.
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if (!busy(n)) continue;
      const int pos = past + shape.depth[node[n]];
      row_lo[n] = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
      int most_lo = row_lo[n];
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) most_lo = max(most_lo, __shfl_xor(most_lo, d));
      wave_lo = max(wave_lo, most_lo);
      float most = 0.0f;
      if (a.q_norm) {
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) sum += squares(x[n][g], y[n][g]);
        const float inv = 1.0f / sqrtf(sum32(sum16(sum)) / (float)D + a.eps);
#pragma unroll
        for (int g = 0; g < G; ++g) norm_pairs<D>(x[n][g], y[n][g], a.q_norm, 4 * g + kq, inv);
      }
      if (a.cos) {
#pragma unroll
        for (int g = 0; g < G; ++g) rotate_pairs(x[n][g], y[n][g], a.cos, a.sin, (long)pos * (D / 2) + 4 * (4 * g + kq));
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
                x[n][g] = x[n][g] * a.prescale * a.qscale;
        y[n][g] = y[n][g] * a.prescale * a.qscale;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = fabsf(x[n][g][i]), w = fabsf(y[n][g][i]);
          most = fmaxf(most, fmaxf(u <= 3.402823466e38f ? u : 0.0f, w <= 3.402823466e38f ? w : 0.0f));
        }
      }
      const unsigned bits = scale_to(max32(max16(most)), 9);
      const float scale = unbits(bits);
      inv_q[n] = inverse_scale(bits);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float v[8] = {x[n][g][0] * scale, x[n][g][1] * scale, x[n][g][2] * scale, x[n][g][3] * scale,
                            y[n][g][0] * scale, y[n][g][1] * scale, y[n][g][2] * scale, y[n][g][3] * scale};
        split8(v, minus_one, &qh[n][g], &ql[n][g]);
      }
    }
  }

  f32x4 o[NB][DT];
  float m[NB], l[NB];  // m: the largest score so far, or up to 7 below it
  bool poison[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = NEG_INF;
    l[n] = 0.0f;
    poison[n] = false;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[n][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  auto compute = [&](int tile, bool bad) __attribute__((always_inline)) {
    const int buf = tile & 1;
    const bool own = tile >= cached;
    const int base = lo + tile * BN;
    f32x4 sc[NB][KBW];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < KBW; ++k) sc[n][k] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int at = (kw * KBW * G + g) * 64 + kq * 16 + ((col ^ (4 * g + kq)) & 15);
      half8 fh[KBW], fl[KBW];
#pragma unroll
      for (int k = 0; k < KBW; ++k) {
        fh[k] = kp_lds[buf][0][k * G * 64 + at];
        fl[k] = kp_lds[buf][1][k * G * 64 + at];
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < KBW; ++k) sc[n][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[k], qh[n][g], sc[n][k], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < KBW; ++k) sc[n][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[k], ql[n][g], sc[n][k], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < KBW; ++k) sc[n][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[k], qh[n][g], sc[n][k], 0, 0, 0);
    }
    const bool hidden = own || bad || base + BN > past || base < wave_lo;
    half8 ph[NB][VBW], pl[NB][VBW];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      // (finite and above 0: hidden scores stay -inf)
      const float f = fminf(fmaxf(inv_q[n] * inverse_scale(kbits), 1.1754944e-38f), 3.402823466e38f);
      if (hidden) {
#pragma unroll
        for (int v = 0; v < VBW; ++v) {
          const int first = 32 * (kw * VBW + v);  // of the tile
          unsigned seen;
          if (own) {
            const int w = ((tile - cached) * BN + first) / 32;
            seen = w < kMaskWords && w * 32 < nodes ? shape.mask[node[n]][w] : 0u;
          } else {
            const int from = max(0, row_lo[n] - base - first), to = min(32, past - base - first);
            seen = from >= 32 || to <= from ? 0u : (0xffffffffu << from) & (0xffffffffu >> (32 - to));
          }
          if (bad) poison[n] |= (seen & bad_lds[kw * VBW + v]) != 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(seen >> ((i & 3) + 4 * kq + 16 * (i >> 2)) & 1u)) sc[n][2 * v + (i >> 2)][i & 3] = NEG_INF;
        }
      }
      float big = NEG_INF;
#pragma unroll
      for (int k = 0; k < KBW; ++k) big = fmaxf(big, fmaxf(fmaxf(sc[n][k][0], sc[n][k][1]), fmaxf(sc[n][k][2], sc[n][k][3])));
      big = max32(max16(big)) * f;
      if (__any(big > m[n] + 7.0f)) {
        const float next = big > m[n] + 7.0f ? big : m[n], keep = fast_exp2(m[n] - safe_max(next));
        m[n] = next;
        l[n] *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] *= keep;
      }
      const float off = 8.0f - safe_max(m[n]);  // weights times 2^8, up to 2^15
#pragma unroll
      for (int v = 0; v < VBW; ++v) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = fast_exp2(fmaf(sc[n][2 * v + (i >> 2)][i & 3], f, off));
          l[n] += p[i];
        }
        split8(p, minus_one, &ph[n][v], &pl[n][v]);
      }
    }
#pragma unroll
    for (int v = 0; v < VBW; ++v)
#pragma unroll
      for (int d = 0; d < DT; d += 4) {
        half8 fh[4], fl[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = ((kw * VBW + v) * DT + d + j) * 64 + kq * 16 + (col ^ j);
          fh[j] = vp_lds[buf][0][at];
          fl[j] = vp_lds[buf][1][at];
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[j], ph[n][v], o[n][d + j], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[j], pl[n][v], o[n][d + j], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[j], ph[n][v], o[n][d + j], 0, 0, 0);
        }
      }
  };

  constexpr unsigned kInfinite = 0x7f800000u;
  constexpr unsigned kTop = (127u + 15u) << 23;  // 2^15
  // Between two barriers a wave computes its part of a tile and writes its share of the
  // next one, the first four waves in the other order: a SIMD has one of each. A tile
  // that has to be written again takes a turn of its own, one in which something is not
  // finite two, as the largest of the rest is not known before it is written. In the
  // first turn there is nothing to compute, and the scales are set between reading the
  // tile's largest and writing it. (Two loops, one for either kind of wave: in one the
  // registers of a tile on its way would be copied, that is waited for.)
  auto turns = [&](auto values) __attribute__((always_inline)) {
    constexpr bool V = decltype(values)::value;
    bool bad = false, rescale = false;
#pragma unroll 1
    for (int tile = t0 - 1; tile < t1;) {
      // (addresses anew each time: kept, they would not leave room for the rest)
      asm volatile("" : "+v"(thread_key), "+v"(thread_channel), "+v"(kl), "+v"(vl), "+v"(vb0), "+v"(vq), "+v"(col), "+v"(kq));
      bool again = false;
      if (tile >= t0) {
        const unsigned km = largest(tile & 1, 4), vm = largest(tile & 1, 0);
        const bool more = km >= kInfinite || vm >= kInfinite;
        // (the largest times the scale, by exponents: bits of both less the bias)
        again = more || rescale || km > kTop - kbits + (127u << 23) || vm > kTop - vbits + (127u << 23);
        if (again) {
          load(tile, values);
          if (more) {
            bad = rescale = true;
            if (tid < VB) bad_lds[tid] = 0;
          } else {
            rescale = false;
            kbits = scale_to(unbits(km), 11);
            unsigned now = scale_to(unbits(vm), 11);
            if (tile > t0) now = min(now, vbits);  // (the output so far only ever gets smaller)
            const float keep = unbits(now) * inverse_scale(vbits);
            vbits = now;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
              for (int d = 0; d < DT; ++d) o[n][d] *= keep;
          }
          __syncthreads();  // (the tile's largest is read, its bad keys cleared)
        }
      }
      const int target = again ? tile : tile + 1;
      const bool computes = tile >= t0 && !again && busy(0);
      if (!V && computes) compute(tile, bad);
      if (target < t1) {
        f32x4 cur[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cur[i] = raw[i];
        if (target >= cached) finish(target, values, cur);
        if (again && bad) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            bool wrong = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bool fine = fabsf(cur[i][j]) < __builtin_inff();
              cur[i][j] = fine ? cur[i][j] : 0.0f;
              wrong |= !fine;
            }
            const int key = thread_key + step_key(i, values);
            if (wrong) atomicOr(&bad_lds[key >> 5], 1u << (key & 31));
          }
        }
        post(target & 1, cur);
        if (tile < t0) {
          __syncthreads();
          kbits = scale_to(unbits(min(largest(t0 & 1, 4), kInfinite - 1)), 11);
          vbits = scale_to(unbits(min(largest(t0 & 1, 0), kInfinite - 1)), 11);
        }
        write(target & 1, values, cur);
      }
      if (target + 1 < t1) {
        load(target + 1, values);
      } else {  // (what the registers hold is of no use: nothing to keep across the turn)
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "=v"(raw[i]));
      }
      if (V && computes) compute(tile, bad);
      if (!again) {
        bad = false;
        ++tile;
      }
      __syncthreads();
    }
  };
  if (values) turns(std::true_type{});
  else turns(std::false_type{});

  // The halves meet: waves 4..7 leave theirs in LDS.
  constexpr int PER = 16 * D + 32;  // floats a block of rows: outputs, scores and sums
  static_assert(KW == 1 || 4 * NB * PER * 4 <= (int)sizeof pieces_lds, "the halves' room");
  float *const room = reinterpret_cast<float *>(pieces_lds);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (!busy(n)) continue;
    l[n] = sum32(sum16(l[n]));
    if (poison[n]) l[n] = __builtin_nanf("");
    if (KW == 2 && kw == 1) {
      float *const mine = room + (rw * NB + n) * PER;
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(mine + d * 256 + lane * 4) = o[n][d];
      if (kq == 0) *reinterpret_cast<float2 *>(mine + 16 * D + 2 * col) = make_float2(m[n], l[n]);
    }
  }
  if (KW == 2) {
    __syncthreads();
    if (kw == 1) return;
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (!busy(n)) continue;
    if (KW == 2) {
      const float *const other = room + (rw * NB + n) * PER;
      const float2 ml = *reinterpret_cast<const float2 *>(other + 16 * D + 2 * col);
      const float big = fmaxf(m[n], ml.x), mine = fast_exp2(m[n] - safe_max(big)), theirs = fast_exp2(ml.x - safe_max(big));
      m[n] = big;
      l[n] = l[n] * mine + ml.y * theirs;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[n][d] = o[n][d] * mine + *reinterpret_cast<const f32x4 *>(other + d * 256 + lane * 4) * theirs;
    }
    const float inv = l[n] == 0.0f ? 0.0f : inverse_scale(vbits) / l[n];
    float *const out = a.splits > 1 ? part(n) : a.out + orow[n] * D;
    if (live[n]) {
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(out + 16 * d + 4 * kq) = o[n][d] * inv;
      if (a.splits > 1) {
        if (kq == 0) *reinterpret_cast<float2 *>(out + D) = make_float2(m[n], l[n]);
      } else if (!(l[n] > 0.0f) || l[n] > 3.402823466e38f) {
        atomicOr(a.err, kDevErrSoftmaxDenominator);
      }
    }
  }
}

// The bf16 prefill operands of the nodes' rows, from the cache's.
// Grid: (blocks over nodes * D, KV heads, sequences), 256 threads.
template <int MB>
__global__ __launch_bounds__(256) void tree_operands_kernel(const TreeArgsOf<MB> a, int D) {
  const int b = blockIdx.z, h = blockIdx.y, at = blockIdx.x * 256 + threadIdx.x, t = at / D, c = at - t * D;
  bf16 *const kb = a.seq[b].kb, *const vt = a.seq[b].vt;
  if (!kb || t >= a.seq[b].nodes) return;
  const long row = a.seq[b].past + t, cap = a.seq[b].cap, from = (row * a.Hkv + h) * D + c;
  kb[((long)h * cap + row) * D + c] = (bf16)a.seq[b].k[from];
  vt[((long)h * D + c) * cap + vt_key_slot(row)] = (bf16)a.seq[b].v[from];
}

// The splits' outputs, each divided by its own sum, by their sums' shares. D / 4
// threads an output row and as many lanes over the splits as a workgroup has room for.
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeMerge a) {
  constexpr int TR = D / 4, SL = 256 / TR, AT_ONCE = 8;
  __shared__ float4 acc_lds[SL][TR];
  __shared__ float2 ml_lds[SL];
  const int c = threadIdx.x % TR, sl = threadIdx.x / TR;
  const long row = blockIdx.x;
  float m = NEG_INF, l = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = sl; i < a.splits; i += SL * AT_ONCE) {
    float2 ml[AT_ONCE];
    float4 x[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const float *const part = a.part + ((long)min(i + j * SL, a.splits - 1) * a.total + row) * (D + 4);
      ml[j] = *reinterpret_cast<const float2 *>(part + D);
      x[j] = reinterpret_cast<const float4 *>(part)[c];
    }
    float big = m;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (i + j * SL >= a.splits) ml[j] = make_float2(NEG_INF, 0.0f);
      big = fmaxf(big, ml[j].x);
    }
    const float keep = fast_exp2(m - safe_max(big));
    l *= keep;
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (ml[j].x == NEG_INF && ml[j].y == 0.0f) continue;  // (a part without keys is not written)
      const float w = ml[j].y * fast_exp2(ml[j].x - safe_max(big));
      l += w;
      acc = make_float4(fmaf(x[j].x, w, acc.x), fmaf(x[j].y, w, acc.y), fmaf(x[j].z, w, acc.z), fmaf(x[j].w, w, acc.w));
    }
    m = big;
  }
  acc_lds[sl][c] = acc;
  if (c == 0) ml_lds[sl] = make_float2(m, l);
  __syncthreads();
  if (sl != 0) return;
  float big = NEG_INF;
#pragma unroll
  for (int i = 0; i < SL; ++i) big = fmaxf(big, ml_lds[i].x);
  l = 0.0f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const float w = fast_exp2(ml_lds[i].x - safe_max(big));
    const float4 x = acc_lds[i][c];
    l = fmaf(ml_lds[i].y, w, l);
    acc = make_float4(fmaf(x.x, w, acc.x), fmaf(x.y, w, acc.y), fmaf(x.z, w, acc.z), fmaf(x.w, w, acc.w));
  }
  if (c == 0 && (!(l > 0.0f) || l > 3.402823466e38f)) atomicOr(a.err, kDevErrSoftmaxDenominator);
  const float inv = 1.0f / l;
  *reinterpret_cast<float4 *>(a.out + row * D + 4 * c) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// The number of splits by a model of the launch: rounds of a workgroup a CU, each of a
// start and its tiles, and the merge, which reads each split's output.
TreePlan tree_plan(int D, int R, int Hkv, int window, const int *past, const int *nodes, int B, int cus) {
  const int BN = 8192 / D;
  int tiles[kMaxDecodeBatch], blocks[kMaxDecodeBatch], most = 1, most_rows = 1;
  long rows = 0;
  TreePlan p;
  for (int b = 0; b < B; ++b) {
    tiles[b] = blocks[b] = 0;
    if (!nodes[b]) continue;
    const int lo = window > 0 ? std::max(0, past[b] + 1 - window) : 0;
    tiles[b] = (past[b] - lo + BN - 1) / BN + (nodes[b] + BN - 1) / BN;
    most_rows = std::max(most_rows, nodes[b] * R);
    most = std::max(most, tiles[b]);
    rows += (long)nodes[b] * R * Hkv;
  }
  p.kw = D < 256 && most_rows <= 64 ? 2 : 1;
  const int per = 128 / p.kw;
  for (int b = 0; b < B; ++b) {
    blocks[b] = (nodes[b] * R + per - 1) / per;
    p.blocks = std::max(p.blocks, blocks[b]);
  }
  constexpr double kStart = 6.0, kTile = 2.7;  // us
  double best = 0.0;
  for (int splits = 1; splits <= std::min(most, 128); ++splits) {
    const int tps = (most + splits - 1) / splits;
    if (splits > 1 && (most + tps - 1) / tps != splits) continue;
    long groups = 0;
    for (int b = 0; b < B; ++b) groups += (long)((tiles[b] + tps - 1) / tps) * blocks[b] * Hkv;
    const double rounds = (double)((groups + cus - 1) / cus);
    const double merge = splits > 1 ? 2.0 + rows * splits * D * 1.0e-6 : 0.0;  // us: a launch, 4 MB a us
    const double time = rounds * (kStart + tps * kTile) + merge;
    if (splits == 1 || time < best) {
      best = time;
      p.splits = splits;
      p.tps = tps;
    }
  }
  return p;
}

template <int D, int KW, int MB>
static void run_tree(hipStream_t st, const TreeArgsOf<MB> &a, int B) {
  hipLaunchKernelGGL((tree_attend_kernel<D, KW, MB>), dim3(a.Hkv, a.splits, B * a.blocks), dim3(512), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(tree_merge_kernel<D>, dim3((unsigned)a.total), dim3(256), 0, st,
                       TreeMerge{a.part, a.out, a.err, a.splits, a.total});
}

template <int MB>
static hipError_t run_tree(hipStream_t st, const TreeArgsOf<MB> &a, int D, int B) {
  if (D == 64 && a.kw == 1) run_tree<64, 1>(st, a, B);
  else if (D == 64) run_tree<64, 2>(st, a, B);
  else if (D == 128 && a.kw == 1) run_tree<128, 1>(st, a, B);
  else if (D == 128) run_tree<128, 2>(st, a, B);
  else run_tree<256, 1>(st, a, B);
  int most = 0;
  for (int b = 0; b < B; ++b)
    if (a.seq[b].kb) most = std::max(most, a.seq[b].nodes);
  if (most) hipLaunchKernelGGL(tree_operands_kernel<MB>, dim3((most * D + 255) / 256, a.Hkv, B), dim3(256), 0, st, a, D);
  return hipGetLastError();
}

hipError_t launch_tree(hipStream_t st, const TreeArgs &a, int D, int B) {
  if (B > 1) return run_tree(st, a, D, B);
  TreeArgsOf<1> one;  // (a launch's arguments cost the host time)
  static_cast<TreeBase &>(one) = a;
  one.seq[0] = a.seq[0];
  return run_tree(st, one, D, 1);
}

// The walk along confirmed nodes: every node that holds the token sampled at its
// parent offers itself as the parent's next, the lowest one stays, and one thread
// follows them. Bound by latency: a load, an LDS read a node of the path, a store.
// Grid: sequences; a wave each.
__global__ __launch_bounds__(64) void tree_accept_kernel(const TreeAcceptArgs a) {
  __shared__ int sampled[kTreeMaxNodes], next[kTreeMaxNodes], path[kTreeMaxNodes];
  const int n = a.nodes[blockIdx.x], lane = threadIdx.x;
  const long first = a.first[blockIdx.x];
  if (n == 0) {
    if (lane == 0) {
      a.count[blockIdx.x] = 0;
      a.next[blockIdx.x] = -1;
    }
    return;
  }
  constexpr int PER = kTreeMaxNodes / 64;
  int parent[PER], token[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = lane + 64 * i;
    if (t < n) {
      sampled[t] = a.sampled[first + t];
      token[i] = a.tokens[first + t];
      parent[i] = a.parents[first + t];
      next[t] = n;
      path[t] = -1;
      if (parent[i] < -1 || parent[i] >= t) {
        atomicOr(a.err, kDevErrTreeParent);
        parent[i] = -1;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = lane + 64 * i;
    if (t < n && parent[i] >= 0) {
      const int want = sampled[parent[i]];
      if (want >= 0 && want == token[i]) atomicMin(&next[parent[i]], t);
    }
  }
  __syncthreads();
  if (lane == 0) {
    int count = 0, last = 0;
    for (int t = 0; t < n; t = next[t]) {  // (a child comes after its parent, so the walk ends)
      path[count++] = t;
      last = t;
    }
    a.count[blockIdx.x] = count;
    a.next[blockIdx.x] = sampled[last];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < n) a.path[first + lane + 64 * i] = path[lane + 64 * i];
}

hipError_t launch_tree_accept(hipStream_t st, const TreeAcceptArgs &a, int B) {
  hipLaunchKernelGGL(tree_accept_kernel, dim3(B), dim3(64), 0, st, a);
  return hipGetLastError();
}

namespace {

// A thread's pieces of rows path[0..n) to rows 0..n. A path rises, so row i is no
// source of a later one, and eight rows at a time are loaded before any is stored.
template <class T, class At>
__device__ __forceinline__ void move_rows(const int *path, int n, At at) {
  for (int i = 0; i < n; i += 8) {
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) v[j] = *reinterpret_cast<const T *>(at(path[i + j]));
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n && path[i + j] != i + j) *reinterpret_cast<T *>(at(i + j)) = v[j];
  }
}

}  // namespace

// Grid: (blocks over a row's pieces, caches, keys or values), 256 threads. Bound by
// latency: the path, then one round of loads and one of stores.
__global__ __launch_bounds__(256) void keep_kernel(const KeepArgs a) {
  __shared__ int path[kTreeMaxNodes], end;
  const KeepCache &c = a.cache[blockIdx.y];
  const bool values = blockIdx.z != 0;
  const int nodes = c.nodes, first = c.first, heads = c.heads, dim = c.dim, kind = c.kind;
  const long cap = c.cap, P = c.past, width = (long)heads * dim;
  char *const rows = values ? +c.v : +c.k, *const more = values ? +c.vp : +c.kp;
  const int t = threadIdx.x;
  int count = a.count[c.seq];
  bool wrong = count < 0 || count > nodes;
  count = min(max(count, 0), nodes);
  if (t == 0) end = count;
  __syncthreads();
  if (t < count) {
    const int p = a.path[first + t];
    path[t] = p;
    if (p < 0 || p >= nodes || (t > 0 && p <= a.path[first + t - 1])) {
      wrong = true;
      atomicMin(&end, t);
    }
  }
  if (wrong && blockIdx.x == 0 && !values) atomicOr(a.err, kDevErrTreePath);
  __syncthreads();
  const int n = end;
  const long unit = (long)blockIdx.x * 256 + t;
  if (kind == 2) {
    // pieces of a head's codes, then its words of step and minimum
    const int pieces = dim / 32, words = dim / 32;
    const long h = unit / (pieces + words);
    const int i = (int)(unit - h * (pieces + words));
    if (h >= heads) return;
    if (i < pieces) {
      char *const p = rows + (h * cap + P) * (dim / 2) + i * 16;
      move_rows<u32x4>(path, n, [&](int r) __attribute__((always_inline)) { return p + (long)r * (dim / 2); });
    } else {
      char *const p = more + ((h * cap + P) * words + (i - pieces)) * 4;
      move_rows<unsigned>(path, n, [&](int r) __attribute__((always_inline)) { return p + (long)r * words * 4; });
    }
    return;
  }
  const bool wide = width % 4 == 0;
  if (unit < (wide ? width / 4 : width)) {
    char *const p = rows + (P * width + unit * (wide ? 4 : 1)) * 4;
    if (wide) move_rows<u32x4>(path, n, [&](int r) __attribute__((always_inline)) { return p + (long)r * width * 4; });
    else move_rows<unsigned>(path, n, [&](int r) __attribute__((always_inline)) { return p + (long)r * width * 4; });
  }
  if (kind == 0) return;
  if (!values) {  // bf16 keys [H, cap, D], eight a thread
    const long h = unit / (dim / 8);
    const int i = (int)(unit - h * (dim / 8));
    if (h >= heads) return;
    char *const p = more + ((h * cap + P) * dim + i * 8) * 2;
    move_rows<u32x4>(path, n, [&](int r) __attribute__((always_inline)) { return p + (long)r * dim * 2; });
  } else {  // bf16 values [H, D, cap], four channels a thread
    for (long i = unit * 4; i < min(unit * 4 + 4, width); ++i) {
      char *const p = more + i * cap * 2;
      move_rows<unsigned short>(path, n, [&](int r) __attribute__((always_inline)) { return p + vt_key_slot(P + r) * 2; });
    }
  }
}

hipError_t launch_keep(hipStream_t st, const KeepArgs &a, int n) {
  long units = 1;
  for (int i = 0; i < n; ++i) {
    const KeepCache &c = a.cache[i];
    const long width = (long)c.heads * c.dim;
    const long u = c.kind == 2 ? width / 16 : width % 4 == 0 ? width / 4 : width;
    units = u > units ? u : units;
  }
  hipLaunchKernelGGL(keep_kernel, dim3((unsigned)((units + 255) / 256), n, 2), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace spissa
