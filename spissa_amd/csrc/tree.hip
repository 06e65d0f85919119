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

// The nodes' depths and, with MASKS, the nodes that each sees, by doubling: after k
// rounds a node knows the 2^k nodes above it. A parent out of its range counts as
// none. For kTreeMaxNodes threads or more; ends with the shape in LDS, after a barrier.
struct TreeShape {
  int depth[kTreeMaxNodes];
  int above[kTreeMaxNodes];  // the node 2^k above
  unsigned mask[kTreeMaxNodes][kMaskWords];
};
// p: the thread's node's parent.
__device__ __forceinline__ void tree_shape(int p, int nodes, int window, bool masks, TreeShape &s, int *err) {
  const int t = threadIdx.x;
  const bool mine = t < nodes;
  if (mine && (p < -1 || p >= t)) {
    if (err) atomicOr(err, kDevErrTreeParent);
    p = -1;
  }
  int depth = p >= 0 ? 1 : 0;
  const int words = (nodes + 31) / 32;
  if (mine && masks)
    for (int w = 0; w < words; ++w) s.mask[t][w] = t >> 5 == w ? 1u << (t & 31) : 0u;
  for (;;) {
    if (mine) {
      s.depth[t] = depth;
      s.above[t] = p;
    }
    if (!__syncthreads_or(p >= 0)) break;
    int up = -1;
    unsigned m[kMaskWords];
    if (p >= 0) {
      depth += s.depth[p];
      up = s.above[p];
      if (masks) {
#pragma unroll
        for (int w = 0; w < kMaskWords; ++w)
          if (w < words) m[w] = s.mask[t][w] | s.mask[p][w];
      }
    }
    __syncthreads();
    if (p >= 0 && masks) {
#pragma unroll
      for (int w = 0; w < kMaskWords; ++w)
        if (w < words) s.mask[t][w] = m[w];
    }
    p = up;
  }
  if (masks && window > 0) {
    if (mine && depth >= window)
      for (int j = 0; j < t; ++j)
        if (depth - s.depth[j] >= window) s.mask[t][j >> 5] &= ~(1u << (j & 31));
    __syncthreads();
  }
}

__device__ __forceinline__ float unbits(unsigned b) { return __uint_as_float(b); }

// Channels 4 l..4 l + 3 and their rotation's partners, half a row on, of row `row`.
template <int D>
__device__ __forceinline__ void load_pairs(const float *row, int l, float4 &lo, float4 &hi) {
  lo = *reinterpret_cast<const float4 *>(row + 4 * l);
  hi = *reinterpret_cast<const float4 *>(row + D / 2 + 4 * l);
}
// The norm's weights times 1 / rms on such channels.
template <int D>
__device__ __forceinline__ void norm_pairs(float4 &lo, float4 &hi, const float *w, int l, float inv) {
#pragma clang fp contract(off)
  float4 a, b;
  load_pairs<D>(w, l, a, b);
  lo = make_float4(lo.x * inv * a.x, lo.y * inv * a.y, lo.z * inv * a.z, lo.w * inv * a.w);
  hi = make_float4(hi.x * inv * b.x, hi.y * inv * b.y, hi.z * inv * b.z, hi.w * inv * b.w);
}
__device__ __forceinline__ void rotate_pairs(float4 &lo, float4 &hi, const float *cos, const float *sin, long at) {
  const float4 c = *reinterpret_cast<const float4 *>(cos + at), s = *reinterpret_cast<const float4 *>(sin + at);
  rotate_pair(lo.x, hi.x, c.x, s.x);
  rotate_pair(lo.y, hi.y, c.y, s.y);
  rotate_pair(lo.z, hi.z, c.z, s.z);
  rotate_pair(lo.w, hi.w, c.w, s.w);
}
__device__ __forceinline__ float squares(const float4 &a, const float4 &b) {
#pragma clang fp contract(off)
  return ((a.x * a.x + b.x * b.x) + (a.y * a.y + b.y * b.y)) + ((a.z * a.z + b.z * b.z) + (a.w * a.w + b.w * b.w));
}

}  // namespace

// Eight waves, each with 16 rows of a KV head (a row: a node and one of the head's
// query heads) and a share of the loads. Keys go by in tiles of 8192 / D: first the
// cached rows from the first that any node sees, then the nodes' own. A tile comes
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
// Grid: (KV heads, splits, sequences x blocks of 128 rows).
template <int D, int MB>
__global__ __launch_bounds__(512, 2) void tree_attend_kernel(const TreeArgsOf<MB> a) {
  constexpr int BN = 8192 / D, G = D / 32, DT = D / 16, VB = BN / 32, KB = BN / 16, TR = D / 8;
  __shared__ __attribute__((aligned(16))) half8 kp_lds[2][2][KB * G * 64];
  __shared__ __attribute__((aligned(16))) half8 vp_lds[2][2][VB * DT * 64];
  __shared__ TreeShape shape;
  __shared__ unsigned most_lds[2][8];
  __shared__ unsigned bad_lds[VB];

  float minus_one = -1.0f;
  asm volatile("" : "+s"(minus_one));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const int h = blockIdx.x, split = blockIdx.y, b = blockIdx.z / a.blocks, block = blockIdx.z - b * a.blocks;
  const int past = a.seq[b].past, nodes = a.seq[b].nodes, seq_first = a.seq[b].first;
  const int rows = nodes * a.R, row0 = block * 128 + wave * 16;
  if (block * 128 >= rows) return;
  const int lo = a.window > 0 ? max(0, past + 1 - a.window) : 0;
  const int cached = (past - lo + BN - 1) / BN, tiles = cached + (nodes + BN - 1) / BN;
  const int t0 = split * a.tps, t1 = min(tiles, t0 + a.tps);

  const int r = min(row0 + col, rows - 1), node = r / a.R, hq = h * a.R + (r - node * a.R);
  const bool live = row0 + col < rows;
  const long orow = (long)(seq_first + node) * a.Hq + hq;
  float *const part = a.part + ((long)split * a.total + orow) * (D + 4);
  if (t0 >= t1) {  // (no keys: nothing of the row's part is read)
    if (live && kq == 0) *reinterpret_cast<float2 *>(part + D) = make_float2(NEG_INF, 0.0f);
    return;
  }

  // A thread's share of a tile: of values eight keys (4 q + 0..3 and 16 + 4 q + 0..3 of
  // 32) of four channels; of keys, four rows' channels 4 l.. and D / 2 + 4 l... Load i
  // has the key thread_key + step_key(i).
  const bool values = wave < 4;
  const int part_of = tid & 255;
  const int vg = part_of / (D / 4);
  int vl = part_of % (D / 4), vb0 = vg >> 2, vq = vg & 3;
  int kl = part_of % TR, kk = part_of / TR;
  int thread_key = values ? vb0 * 32 + 4 * vq : kk, thread_channel = values ? 4 * vl : 4 * kl;
  const long stride = (long)a.Hkv * D;
  float *const cache_rows = (values ? +a.seq[b].v : +a.seq[b].k) + h * D;
  const float *const own_rows = (values ? +a.v : +a.k) + seq_first * stride + h * D;
  bf16 *const kb = a.seq[b].kb, *const vt = a.seq[b].vt;
  const long cap = a.seq[b].cap;
  float4 raw[8];
  auto step_key = [&](int i) __attribute__((always_inline)) { return values ? (i & 3) + 16 * (i >> 2) : (i >> 1) * (256 / TR); };
  auto load = [&](int tile) __attribute__((always_inline)) {
    const bool own = tile >= cached;
    const int first = own ? (tile - cached) * BN : lo + tile * BN, left = (own ? nodes : past) - first;
    const char *const src = reinterpret_cast<const char *>((own ? own_rows : +cache_rows) + first * stride);
    if (left >= BN) {
      const unsigned off = (unsigned)(thread_key * stride + thread_channel) * 4u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        raw[i] = *reinterpret_cast<const float4 *>(src + (step_key(i) * stride + (values ? 0 : (i & 1) * (D / 2))) * 4 + off);
    } else {  // (rows past the last: that one again)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long at = min(thread_key + step_key(i), left - 1) * stride + thread_channel + (values ? 0 : (i & 1) * (D / 2));
        raw[i] = *reinterpret_cast<const float4 *>(src + at * 4);
      }
    }
  };
  // The nodes' own rows: the norm and the rotation of keys, and the append.
  auto finish = [&](int tile) __attribute__((always_inline)) {
    const int first = (tile - cached) * BN + thread_key;
    if (!values) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int t = min(first + step_key(i), nodes - 1);
        if (a.k_norm) {
          const float inv = 1.0f / sqrtf(group_sum<TR>(squares(raw[i], raw[i + 1])) / (float)D + a.eps);
          norm_pairs<D>(raw[i], raw[i + 1], a.k_norm, kl, inv);
        }
        if (a.cos) rotate_pairs(raw[i], raw[i + 1], a.cos, a.sin, (long)(past + shape.depth[t]) * (D / 2) + 4 * kl);
      }
    }
    if (block != 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = first + step_key(i);
      if (t >= nodes) continue;
      const long at = past + t;
      const int c = thread_channel + (values ? 0 : (i & 1) * (D / 2));
      *reinterpret_cast<float4 *>(cache_rows + at * stride + c) = raw[i];
      if (!kb) continue;
      const float x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      bf16 *const dst = values ? vt + ((long)h * D + c) * cap + vt_key_slot(at) : kb + ((long)h * cap + at) * D + c;
      const long step = values ? cap : 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[j * step] = (bf16)x[j];
    }
  };
  // The wave's largest magnitude, as bits (a NaN or an infinity is above the rest).
  auto post = [&](int slot) __attribute__((always_inline)) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = max(m, max(__float_as_uint(raw[i].x) & 0x7fffffffu, __float_as_uint(raw[i].y) & 0x7fffffffu));
      m = max(m, max(__float_as_uint(raw[i].z) & 0x7fffffffu, __float_as_uint(raw[i].w) & 0x7fffffffu));
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, d));
    if (lane == 0) most_lds[slot][wave] = m;
  };
  unsigned kbits = 127u << 23, vbits = 127u << 23;  // the scales, as float bits
  auto write = [&](int buf) __attribute__((always_inline)) {
    const float scale = unbits(values ? vbits : kbits);
    if (values) {
      const int dt = vl >> 2;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (c == 0 ? raw[i].x : c == 1 ? raw[i].y : c == 2 ? raw[i].z : raw[i].w) * scale;
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
        const float v[8] = {raw[i].x * scale,     raw[i].y * scale,     raw[i].z * scale,     raw[i].w * scale,
                            raw[i + 1].x * scale, raw[i + 1].y * scale, raw[i + 1].z * scale, raw[i + 1].w * scale};
        half8 ph, pl;
        split8(v, minus_one, &ph, &pl);
        const int key = thread_key + step_key(i), at = ((key >> 4) * G + (kl >> 2)) * 64 + (kl & 3) * 16 + ((key ^ kl) & 15);
        kp_lds[buf][0][at] = ph;
        kp_lds[buf][1][at] = pl;
      }
    }
  };
  auto largest = [&](int slot, int from) __attribute__((always_inline)) {
    const unsigned *m = most_lds[slot] + from;
    return max(max(m[0], m[1]), max(m[2], m[3]));
  };

  // (all that needs no other load first: the parents, the queries, the first tiles)
  const int parent = tid < nodes ? a.parents[seq_first + tid] : -1;
  float4 x[G], y[G];
#pragma unroll
  for (int g = 0; g < G; ++g) load_pairs<D>(a.q + orow * D, 4 * g + kq, x[g], y[g]);
  load(t0);
  tree_shape(parent, nodes, a.window, t1 > cached, shape, block == 0 && split == 0 && h == 0 ? a.err : nullptr);

  // The queries of the wave's rows, as the B operand.
  half8 qh[G], ql[G];
  float inv_q;
  const int pos = past + shape.depth[node], row_lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  {
    float most = 0.0f;
    if (a.q_norm) {
      float sum = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) sum += squares(x[g], y[g]);
      const float inv = 1.0f / sqrtf(sum32(sum16(sum)) / (float)D + a.eps);
#pragma unroll
      for (int g = 0; g < G; ++g) norm_pairs<D>(x[g], y[g], a.q_norm, 4 * g + kq, inv);
    }
    if (a.cos) {
#pragma unroll
      for (int g = 0; g < G; ++g) rotate_pairs(x[g], y[g], a.cos, a.sin, (long)pos * (D / 2) + 4 * (4 * g + kq));
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float *const v[8] = {&x[g].x, &x[g].y, &x[g].z, &x[g].w, &y[g].x, &y[g].y, &y[g].z, &y[g].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        *v[i] = *v[i] * a.prescale * a.qscale;
        const float m = fabsf(*v[i]);
        most = fmaxf(most, m <= 3.402823466e38f ? m : 0.0f);
      }
    }
    const unsigned bits = scale_to(max32(max16(most)), 9);
    const float scale = unbits(bits);
    inv_q = inverse_scale(bits);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float v[8] = {x[g].x * scale, x[g].y * scale, x[g].z * scale, x[g].w * scale,
                          y[g].x * scale, y[g].y * scale, y[g].z * scale, y[g].w * scale};
      split8(v, minus_one, &qh[g], &ql[g]);
    }
  }
  int wave_lo = row_lo;  // keys from here on are seen by all rows of the wave
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) wave_lo = max(wave_lo, __shfl_xor(wave_lo, d));

  f32x4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, l = 0.0f;  // m: the largest score so far, or up to 7 below it
  bool poison = false;

  auto compute = [&](int tile, bool bad) __attribute__((always_inline)) {
    const int buf = tile & 1;
    const bool own = tile >= cached;
    const int base = lo + tile * BN;
    f32x4 sc[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) sc[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int at = g * 64 + kq * 16 + ((col ^ (4 * g + kq)) & 15);
      half8 fh[KB], fl[KB];
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        fh[k] = kp_lds[buf][0][k * G * 64 + at];
        fl[k] = kp_lds[buf][1][k * G * 64 + at];
      }
#pragma unroll
      for (int k = 0; k < KB; ++k) sc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[k], qh[g], sc[k], 0, 0, 0);
#pragma unroll
      for (int k = 0; k < KB; ++k) sc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[k], ql[g], sc[k], 0, 0, 0);
#pragma unroll
      for (int k = 0; k < KB; ++k) sc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[k], qh[g], sc[k], 0, 0, 0);
    }
    // (finite and above 0: hidden scores stay -inf)
    const float f = fminf(fmaxf(inv_q * inverse_scale(kbits), 1.1754944e-38f), 3.402823466e38f);
    // (scores of hidden keys at -inf)
    if (own || bad || base + BN > past || base < wave_lo) {
#pragma unroll
      for (int v = 0; v < VB; ++v) {
        unsigned seen;
        if (own) {
          const int w = (tile - cached) * VB + v;
          seen = w < kMaskWords && w * 32 < nodes ? shape.mask[node][w] : 0u;
        } else {
          const int from = max(0, row_lo - base - 32 * v), to = min(32, past - base - 32 * v);
          seen = from >= 32 || to <= from ? 0u : (0xffffffffu << from) & (0xffffffffu >> (32 - to));
        }
        if (bad) poison |= (seen & bad_lds[v]) != 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(seen >> ((i & 3) + 4 * kq + 16 * (i >> 2)) & 1u)) sc[2 * v + (i >> 2)][i & 3] = NEG_INF;
      }
    }
    float big = NEG_INF;
#pragma unroll
    for (int k = 0; k < KB; ++k) big = fmaxf(big, fmaxf(fmaxf(sc[k][0], sc[k][1]), fmaxf(sc[k][2], sc[k][3])));
    big = max32(max16(big)) * f;
    if (__any(big > m + 7.0f)) {
      const float next = big > m + 7.0f ? big : m, keep = fast_exp2(m - safe_max(next));
      m = next;
      l *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= keep;
    }
    const float off = 8.0f - safe_max(m);  // weights times 2^8, up to 2^15
    half8 ph[VB], pl[VB];
#pragma unroll
    for (int v = 0; v < VB; ++v) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = fast_exp2(fmaf(sc[2 * v + (i >> 2)][i & 3], f, off));
        l += p[i];
      }
      split8(p, minus_one, &ph[v], &pl[v]);
    }
#pragma unroll
    for (int v = 0; v < VB; ++v)
#pragma unroll
      for (int d = 0; d < DT; d += 4) {
        half8 fh[4], fl[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = (v * DT + d + j) * 64 + kq * 16 + (col ^ j);
          fh[j] = vp_lds[buf][0][at];
          fl[j] = vp_lds[buf][1][at];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[j], ph[v], o[d + j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[j], pl[v], o[d + j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[j], ph[v], o[d + j], 0, 0, 0);
      }
  };

  constexpr unsigned kInfinite = 0x7f800000u;
  constexpr unsigned kTop = (127u + 15u) << 23;  // 2^15
  // The first tile in LDS, with the scales that it sets.
  if (t0 >= cached) finish(t0);
  post(t0 & 1);
  __syncthreads();
  kbits = scale_to(unbits(min(largest(t0 & 1, 4), kInfinite - 1)), 11);
  vbits = scale_to(unbits(min(largest(t0 & 1, 0), kInfinite - 1)), 11);
  write(t0 & 1);
  if (t0 + 1 < t1) load(t0 + 1);
  __syncthreads();

  // Between two barriers a wave computes its rows' part of a tile and writes its share
  // of the next one, the first four waves in the other order: a SIMD has one of each.
  // A tile that has to be written again takes a turn of its own, one in which something
  // is not finite two, as the largest of the rest is not known before it is written.
  bool bad = false, rescale = false;
#pragma unroll 1
  for (int tile = t0; tile < t1;) {
    // (addresses anew each turn: kept, they would not leave room for the rest)
    asm volatile("" : "+v"(thread_key), "+v"(thread_channel), "+v"(kl), "+v"(vl), "+v"(vb0), "+v"(vq));
    const unsigned km = largest(tile & 1, 4), vm = largest(tile & 1, 0);
    const bool more = km >= kInfinite || vm >= kInfinite;
    // (the largest times the scale, by exponents: bits of both less the bias)
    const bool again = more || rescale || km > kTop - kbits + (127u << 23) || vm > kTop - vbits + (127u << 23);
    const int target = again ? tile : tile + 1;
    if (again) {
      load(tile);
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
        for (int d = 0; d < DT; ++d) o[d] *= keep;
      }
      __syncthreads();  // (the tile's largest is read, its bad keys cleared)
    }
    auto stage = [&]() __attribute__((always_inline)) {
      if (target >= t1) return;
      if (target >= cached) finish(target);
      if (again && bad) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          bool wrong = false;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!(fabsf(v[j]) < __builtin_inff())) {
              v[j] = 0.0f;
              wrong = true;
            }
          raw[i] = make_float4(v[0], v[1], v[2], v[3]);
          const int key = thread_key + step_key(i);
          if (wrong) atomicOr(&bad_lds[key >> 5], 1u << (key & 31));
        }
      }
      post(target & 1);
      write(target & 1);
      if (target + 1 < t1) load(target + 1);
    };
    if (values) stage();
    if (!again && row0 < rows) compute(tile, bad);
    if (!values) stage();
    if (!again) {
      bad = false;
      ++tile;
    }
    __syncthreads();
  }

  if (row0 >= rows) return;
  l = sum32(sum16(l));
  if (poison) l = __builtin_nanf("");
  const float inv = l == 0.0f ? 0.0f : inverse_scale(vbits) / l;
  float *const out = a.splits > 1 ? part : a.out + orow * D;
  if (live) {
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(out + 16 * d + 4 * kq) = o[d] * inv;
    if (a.splits > 1) {
      if (kq == 0) *reinterpret_cast<float2 *>(part + D) = make_float2(m, l);
    } else if (!(l > 0.0f) || l > 3.402823466e38f) {
      atomicOr(a.err, kDevErrSoftmaxDenominator);
    }
  }
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
  int tiles[kMaxDecodeBatch], blocks[kMaxDecodeBatch], most = 1;
  long rows = 0;
  TreePlan p;
  for (int b = 0; b < B; ++b) {
    tiles[b] = blocks[b] = 0;
    if (!nodes[b]) continue;
    const int lo = window > 0 ? std::max(0, past[b] + 1 - window) : 0;
    tiles[b] = (past[b] - lo + BN - 1) / BN + (nodes[b] + BN - 1) / BN;
    blocks[b] = (nodes[b] * R + 127) / 128;
    most = std::max(most, tiles[b]);
    p.blocks = std::max(p.blocks, blocks[b]);
    rows += (long)nodes[b] * R * Hkv;
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

template <int D, int MB>
static void run_tree(hipStream_t st, const TreeArgsOf<MB> &a, int B) {
  hipLaunchKernelGGL((tree_attend_kernel<D, MB>), dim3(a.Hkv, a.splits, B * a.blocks), dim3(512), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(tree_merge_kernel<D>, dim3((unsigned)a.total), dim3(256), 0, st,
                       TreeMerge{a.part, a.out, a.err, a.splits, a.total});
}

template <int MB>
static hipError_t run_tree(hipStream_t st, const TreeArgsOf<MB> &a, int D, int B) {
  if (D == 64) run_tree<64>(st, a, B);
  else if (D == 128) run_tree<128>(st, a, B);
  else run_tree<256>(st, a, B);
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
