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
constexpr int kTreeRows = 128;  // of a workgroup: a node and one of the KV head's query heads each

// The nodes' depths and, with MASKS, the nodes that each sees (with a window those less
// than it apart), by doubling: after k rounds a node knows the 2^k nodes above it. A
// parent out of its range counts as none. For 256 threads; p: the thread's node's parent.
struct TreeShape {
  int depth[kTreeMaxNodes];
  int above[kTreeMaxNodes];  // the node 2^k above
  unsigned mask[kTreeMaxNodes][kMaskWords];
};
template <bool MASKS>
__device__ __forceinline__ void tree_shape(int p, int nodes, int window, TreeShape &s, int *err) {
  const int t = threadIdx.x;
  if (p < -1 || p >= t) {
    if (err && t < nodes) atomicOr(err, kDevErrTreeParent);
    p = -1;
  }
  int depth = p >= 0 ? 1 : 0;
  unsigned m[kMaskWords];
#pragma unroll
  for (int w = 0; w < kMaskWords; ++w) m[w] = MASKS && t >> 5 == w ? 1u << (t & 31) : 0u;
  for (;;) {
    s.depth[t] = depth;
    s.above[t] = p;
    if (MASKS) {
#pragma unroll
      for (int w = 0; w < kMaskWords; ++w) s.mask[t][w] = m[w];
    }
    if (!__syncthreads_or(p >= 0)) break;
    if (p >= 0) {
      depth += s.depth[p];
      if (MASKS) {
#pragma unroll
        for (int w = 0; w < kMaskWords; ++w) m[w] |= s.mask[p][w];
      }
      p = s.above[p];
    }
    __syncthreads();
  }
  if (MASKS && window > 0 && t < nodes && depth >= window)
    for (int j = 0; j < t; ++j)
      if (depth - s.depth[j] >= window) s.mask[t][j >> 5] &= ~(1u << (j & 31));
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
// The norm's weights times 1 / rms.
__device__ __forceinline__ f32x4 norm4(f32x4 x, f32x4 w, float inv) {
#pragma clang fp contract(off)
  return x * inv * w;
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

// Where the queries of 16 rows are: two pieces of [D / 32][64 lanes], the inverse
// scales and the first keys.
template <int D>
struct TreeQuery {
  char *at;
  __device__ __forceinline__ TreeQuery(char *queries, long group) : at(queries + group * tree_query_bytes(D)) {}
  __device__ __forceinline__ half8 *piece(int which, int g) const {
    return reinterpret_cast<half8 *>(at) + (which * (D / 32) + g) * 64;
  }
  __device__ __forceinline__ float *inverse() const { return reinterpret_cast<float *>(at + 64 * D); }
  __device__ __forceinline__ int *from() const { return reinterpret_cast<int *>(at + 64 * D + 64); }
};

}  // namespace

// Up to 64 nodes, by each wave for itself: lane t's depth and nodes that it sees. (A step
// of 26 nodes 32.4 us, with tree_shape 33.6.)
struct SmallShape {
  int depth;
  unsigned lo, hi;
};
__device__ __forceinline__ SmallShape small_shape(int p, int nodes, int *err) {
  const int t = threadIdx.x & 63;
  if (p < -1 || p >= t) {
    if (err && t < nodes) atomicOr(err, kDevErrTreeParent);
    p = -1;
  }
  SmallShape s{p >= 0 ? 1 : 0, t < 32 ? 1u << t : 0u, t < 32 ? 0u : 1u << (t - 32)};
  while (__any(p >= 0)) {
    const int from = p < 0 ? t : p;
    const int d = __shfl(s.depth, from), up = __shfl(p, from);
    const unsigned l = (unsigned)__shfl((int)s.lo, from), h = (unsigned)__shfl((int)s.hi, from);
    if (p >= 0) {
      s.depth += d;
      s.lo |= l;
      s.hi |= h;
      p = up;
    }
  }
  return s;
}

// What the attention takes of the nodes, once each: the norm and the rotation of queries
// and keys, keys and values into the cache (and its bf16 prefill operands), the queries
// of 16 rows (a row: a node and one of the KV head's query heads; the last 16 are filled
// up with the last row) as the B operand of the scores' product, two binary16 pieces of
// the query times a power of two, the power's inverse, the first key that the row sees,
// and the nodes that a node sees. D / 8 lanes a row, each with four channels and their
// rotation's partners. Bound by latency: the parents, the rotation's rows, the stores
// (5 nodes of 32 + 2 x 8 rows of 64: 4 us; 256 of 4 + 2 x 1 of 256: 8 us; by each attention
// workgroup for itself it cost 16 ragged sequences a quarter of their time).
// Grid: (blocks of rows of the longest sequence, sequences), 256 threads.
template <int D, int MB>
__global__ __launch_bounds__(256) void tree_prepare_kernel(const TreeArgsOf<MB> a) {
  constexpr int TR = D / 8, LINES = 256 / TR;
  __shared__ TreeShape shape;
  const int b = blockIdx.y, past = a.seq[b].past, nodes = a.seq[b].nodes, first = a.seq[b].first;
  const int rows = nodes * a.R, padded = (rows + 15) & ~15;
  const int queries = padded * a.Hkv, lines = queries + nodes * a.Hkv * 2;  // queries, keys, values
  if ((int)blockIdx.x * LINES >= lines) return;
  const int tid = threadIdx.x, lane = tid & 63, l = tid % TR, line = min((int)blockIdx.x * LINES + tid / TR, lines - 1);
  const int parent = nodes <= 64 ? (lane < nodes ? a.parents[first + lane] : -1) : tid < nodes ? a.parents[first + tid] : -1;
  const int kind = line < queries ? 0 : line < queries + nodes * a.Hkv ? 1 : 2;
  const int in = kind == 0 ? line : kind == 1 ? line - queries : line - queries - nodes * a.Hkv;
  // (a KV head's padded rows lie together, a node's heads do)
  const int h = kind == 0 ? in / padded : in % a.Hkv, place = in - h * padded;
  const int row = min(place, rows - 1), node = kind == 0 ? row / a.R : in / a.Hkv;
  const float *const src = kind == 0 ? a.q + ((long)(first + node) * a.Hq + h * a.R + (row - node * a.R)) * D
                                     : (kind == 1 ? +a.k : +a.v) + ((long)first * a.Hkv + in) * D;
  f32x4 x, y, u, w;
  load_pairs<D>(src, l, x, y);
  if (a.q_norm && kind < 2) load_pairs<D>(kind == 0 ? +a.q_norm : +a.k_norm, l, u, w);
  int *const err = blockIdx.x == 0 && tid < 64 ? a.err : nullptr;
  int depth;
  if (nodes <= 64 && !(a.window > 0 && a.window < nodes)) {
    const SmallShape s = small_shape(parent, nodes, err);  // (a window that may part nodes takes the other)
    depth = __shfl(s.depth, node);
    if (blockIdx.x == 0 && tid < nodes) {
      a.mask[(long)(first + tid) * kMaskWords] = s.lo;
      a.mask[(long)(first + tid) * kMaskWords + 1] = s.hi;
    }
  } else {
    const int mine = nodes <= 64 && tid >= 64 ? -1 : parent;
    if (blockIdx.x == 0) {
      tree_shape<true>(mine, nodes, a.window, shape, a.err);
      if (tid < nodes) {
#pragma unroll
        for (int i = 0; i < kMaskWords; ++i) a.mask[(long)(first + tid) * kMaskWords + i] = shape.mask[tid][i];
      }
    } else {
      tree_shape<false>(mine, nodes, a.window, shape, nullptr);
    }
    depth = shape.depth[node];
  }
  if (kind < 2) {
    if (a.q_norm) {
      const float inv = 1.0f / sqrtf(group_sum<TR>(squares(x, y)) / (float)D + a.eps);
      x = norm4(x, u, inv);
      y = norm4(y, w, inv);
    }
    if (a.cos) rotate_pairs(x, y, a.cos, a.sin, (long)(past + depth) * (D / 2) + 4 * l);
  }
  if ((int)blockIdx.x * LINES + tid / TR >= lines) return;
  if (kind == 0) {
    float minus_one = -1.0f;
    asm volatile("" : "+s"(minus_one));
    x = x * a.prescale * a.qscale;
    y = y * a.prescale * a.qscale;
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = fabsf(x[i]), q = fabsf(y[i]);
      most = fmaxf(most, fmaxf(p <= 3.402823466e38f ? p : 0.0f, q <= 3.402823466e38f ? q : 0.0f));
    }
    most = fmaxf(most, dpp<0xB1>(most));
    most = fmaxf(most, dpp<0x4E>(most));
    most = fmaxf(most, dpp<0x141>(most));
    if constexpr (TR >= 16) most = fmaxf(most, dpp<0x140>(most));
    if constexpr (TR >= 32) most = max16(most);
    const unsigned bits = scale_to(most, 9);
    const float scale = unbits(bits);
    const float v[8] = {x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale, y[0] * scale, y[1] * scale, y[2] * scale, y[3] * scale};
    half8 ph, pl;
    split8(v, minus_one, &ph, &pl);
    const TreeQuery<D> out(a.queries, a.seq[b].group0 + (place >> 4) * a.Hkv + h);
    const int at = (l & 3) * 16 + (place & 15);
    out.piece(0, l >> 2)[at] = ph;
    out.piece(1, l >> 2)[at] = pl;
    if (l == 0) {
      out.inverse()[place & 15] = inverse_scale(bits);
      out.from()[place & 15] = a.window > 0 ? max(0, past + depth + 1 - a.window) : 0;
    }
    return;
  }
  const long at = past + node;
  const int head = in % a.Hkv;
  float *const dst = (kind == 1 ? +a.seq[b].k : +a.seq[b].v) + (at * a.Hkv + head) * D + 4 * l;
  *reinterpret_cast<f32x4 *>(dst) = x;
  *reinterpret_cast<f32x4 *>(dst + D / 2) = y;
  bf16 *const kb = a.seq[b].kb, *const vt = a.seq[b].vt;
  if (kb) {
    const long cap = a.seq[b].cap, step = kind == 1 ? 1 : cap;
    bf16 *const to = kind == 1 ? kb + ((long)head * cap + at) * D + 4 * l : vt + ((long)head * D + 4 * l) * cap + vt_key_slot(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      to[i * step] = (bf16)x[i];
      to[(D / 2 + i) * step] = (bf16)y[i];
    }
  }
}

// The unit (KV head of a block of rows of a sequence) that the launch's tile `at` is of.
struct TreeUnit {
  int b, block, h;
  int start, tiles, padded;  // its first place, its tiles, the places that they take
};
template <class Args>
__device__ __forceinline__ TreeUnit tree_unit(const Args &a, int at) {
  TreeUnit u;
  u.b = 0;
  while (u.b < a.B - 1 && at >= a.seq[u.b + 1].start) ++u.b;
  u.tiles = a.seq[u.b].tiles;
  u.padded = a.seq[u.b].padded;
  const int which = (at - a.seq[u.b].start) / u.padded;
  u.block = which / a.Hkv;
  u.h = which - u.block * a.Hkv;
  u.start = a.seq[u.b].start + which * u.padded;
  return u;
}

// Eight waves of 16 rows (a node and one of the KV head's query heads) each, which take
// tiles of 8192 / D keys. Tiles are first the cached rows from the first that any node
// sees, then the nodes' own. A tile comes into registers while the
// one before is computed; waves 0..3 take its values, waves 4..7 its keys, and write
// them to LDS once for all rows as two binary16 pieces, in the order in which lanes take
// the operands. S^T = K Q^T, so a lane has one row (column lane % 16) and four keys of
// each 16, and two such blocks are the B operand of O^T += V^T P^T without an exchange,
// the values' keys being stored in that order. Channels of the scores' product come as
// 4 l..4 l + 3 beside D / 2 + 4 l..., as the rotation pairs them.
//
// Scales. Pieces hold 2^-23 of a number only between 2^-3 and 2^16, and 2^-25 below. Keys
// and values are multiplied by a power of two that takes the first tile's largest to
// 2^11..2^12. Whether a tile's largest number is above 2^15, or eight channels of one of its
// rows all below 2^-2 (and not 0), is known after it is written. Such a tile is loaded and written again with a scale of its own; one whose rows no scale takes
// together (more than 2^13 apart, or one not finite) in parts, from the largest keys
// down, each with zeros in the place of the other rows, which nobody sees in that turn. So
// every row is held to 2^-23 of its own largest, whatever stands beside it. A row with a
// number that is not finite is in no part, but noted: nodes that see it become NaN. (The
// step of 26 nodes below, 33 us: with one value of 1e6 43, with one in every tile 85, with
// rows of 2^-40 to 2^40 182. With a key channel of 400 in every row it stays: of four
// channels instead of eight, all small ones were common, 43 us.)
//
// An output row is held times a power of two, its unit: the values' scale, as long as that
// stays. Where it changes, a row takes the new one unless that costs it what it holds: one
// whose weights are small (or nothing) beside larger values keeps its unit, and one that holds
// large values keeps it where smaller ones follow; their weights are then multiplied by
// what the two differ by.
//
// Work. The launch's units (a KV head of a block of rows of a sequence) lie one after
// the other with their tiles, and a workgroup takes `share` of them in a row, of one
// unit or of several; a unit of several workgroups' is merged by tree_merge_kernel.
//
// Bound by HBM with few rows (a step of 16 sequences of up to 8192 keys, 12 nodes each, 24
// heads on 8 of 128: 145 us, 4.8 TB/s; of one sequence, 26 nodes: 32.5 us, of which 6 fill and
// drain this pipeline and 7 are the other launches, and half a one the smallest channels), by dependent chains of LDS reads and
// matrix instructions at two waves a SIMD with many (256 nodes over 32768 keys, 4 heads on
// one of 256: 130 to 138 us, 250 to 265 TFLOP/s of plain products, three times that of pieces). Two waves
// sharing 16 rows' keys, where half the waves have no rows, came to the same (64 rows over
// 8192 keys of 8 heads of 128: 28.2 us a step against 27.2).
//
// Grid: workgroups.
template <int D, int MB>
__global__ __launch_bounds__(512, 2) void tree_attend_kernel(const TreeArgsOf<MB> a) {
  constexpr int BN = 8192 / D, G = D / 32, DT = D / 16, VB = BN / 32, KB = BN / 16, TR = D / 8;
  constexpr int ROWS = kTreeRows;
  constexpr int AHEAD = 2;  // (three: the same with heads of 64 and 128, a tenth slower with heads of 256)
  static_assert(KB * G == 16 && VB * DT == 16, "a tile has 8192 keys' and as many values' channels");
  __shared__ __attribute__((aligned(16))) half8 pieces_lds[2][2][2][1024];  // values, buffer, piece
  half8 (*const kp_lds)[2][1024] = pieces_lds[0], (*const vp_lds)[2][1024] = pieces_lds[1];
  constexpr int kSpan = 13;  // powers of two between the largest rows of a part and its smallest
  __shared__ __attribute__((aligned(16))) unsigned most_lds[2][8], least_lds[2][8];
  __shared__ __attribute__((aligned(8))) unsigned char unfit_lds[2][8];
  __shared__ unsigned size_lds[2 * BN];  // of a tile in parts: its keys' largest, then its values', as bits
  __shared__ unsigned bad_lds[VB], left_lds[VB], take_lds[VB], scale_lds[3];
  __shared__ int unit_lds[8][16];

  float minus_one = -1.0f;
  asm volatile("" : "+s"(minus_one));
  int place = blockIdx.x * a.share;
  const int end = min(place + a.share, a.places);
#pragma unroll 1
  while (place < end) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (what follows from it is formed in each turn: kept, it would not leave room for the rest)
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int col = lane & 15, kq = lane >> 4;
    const bool values = wave < 4;
    const TreeUnit unit = tree_unit(a, place);
    const int t0 = place - unit.start, t1 = min(unit.tiles, t0 + (end - place));
    const int slot_of = (int)blockIdx.x - unit.start / a.share;
    if (place != (int)blockIdx.x * a.share) __syncthreads();  // (the unit before is done with LDS)
    place = unit.start + unit.padded;
    if (t0 >= t1) continue;
    const int past = a.seq[unit.b].past, nodes = a.seq[unit.b].nodes, rows = nodes * a.R;
    const int lo = a.window > 0 ? max(0, past + 1 - a.window) : 0;
    const int cached = (past - lo + BN - 1) / BN;
    const int row0 = unit.block * ROWS + wave * 16;
    const bool busy = row0 < rows;

    // A thread's share of a tile: of values eight keys (4 q + 0..3 and 16 + 4 q + 0..3 of
    // 32) of four channels; of keys, four rows' channels 4 l.. and D / 2 + 4 l... Load i
    // has the key thread_key + step_key(i).
    const int part_of = tid & 255;
    const int vg = part_of / (D / 4);
    int vl = part_of % (D / 4), vb0 = vg >> 2, vq = vg & 3;
    int kl = part_of % TR, kk = part_of / TR;
    int thread_key = values ? vb0 * 32 + 4 * vq : kk, thread_channel = values ? 4 * vl : 4 * kl;
    const long stride = (long)a.Hkv * D;
    const float *const cache_rows = (values ? +a.seq[unit.b].v : +a.seq[unit.b].k) + unit.h * D;
    f32x4 raw[8];
    auto step_key = [&](int i) __attribute__((always_inline)) { return values ? (i & 3) + 16 * (i >> 2) : (i >> 1) * (256 / TR); };
    auto load = [&](int tile) __attribute__((always_inline)) {
      const bool own = tile >= cached;
      const int first = own ? past + (tile - cached) * BN : lo + tile * BN, last = (own ? past + nodes : past) - first - 1;
      const char *const src = reinterpret_cast<const char *>(cache_rows + first * stride);
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // (rows past the last: that one again)
        const unsigned at = (unsigned)min(thread_key + step_key(i), last) * (unsigned)stride + thread_channel + (values ? 0 : (i & 1) * (D / 2));
        raw[i] = *reinterpret_cast<const f32x4 *>(src + at * 4u);
      }
    };
    auto bits_of = [&](const f32x4 &x) __attribute__((always_inline)) {
      return max(max(__float_as_uint(x[0]) & 0x7fffffffu, __float_as_uint(x[1]) & 0x7fffffffu),
                 max(__float_as_uint(x[2]) & 0x7fffffffu, __float_as_uint(x[3]) & 0x7fffffffu));
    };
    // The wave's largest magnitude, as bits (a NaN or an infinity is above the rest), and
    // the smallest of eight channels' largest less 1 (eight zeros are above the rest).
    auto post = [&](int slot, const f32x4 (&cur)[8]) __attribute__((always_inline)) -> uint2 {
      unsigned m = 0, s = ~0u, of[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        of[i] = bits_of(cur[i]);
        m = max(m, of[i]);
      }
      if (values) {  // (the neighbour has the same keys' next four channels, or the ones before)
#pragma unroll
        for (int i = 0; i < 8; ++i) of[i] = max(of[i], (unsigned)__builtin_amdgcn_update_dpp((int)of[i], (int)of[i], 0xB1, 0xf, 0xf, false));
      } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) of[i] = of[i + 1] = max(of[i], of[i + 1]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s = min(s, of[i] - 1u);
      m = wave_max_bits(m);
      s = ~wave_max_bits(~s);
      if (lane == 0) {
        most_lds[slot][wave] = m;
        least_lds[slot][wave] = s;
      }
      return uint2{m, s};
    };
    unsigned kbits = 127u << 23, vbits = 127u << 23;  // the scales, as float bits
    auto write = [&](int buf, const f32x4 (&cur)[8]) __attribute__((always_inline)) {
      if (values) {
        const float scale = unbits(vbits);
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
        const float scale = unbits(kbits);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float v[8] = {cur[i][0] * scale,     cur[i][1] * scale,     cur[i][2] * scale,     cur[i][3] * scale,
                              cur[i + 1][0] * scale, cur[i + 1][1] * scale, cur[i + 1][2] * scale, cur[i + 1][3] * scale};
          half8 ph, pl;
          split8(v, minus_one, &ph, &pl);
          const int key = thread_key + step_key(i), at = ((key >> 4) * G + (kl >> 2)) * 64 + (kl & 3) * 16 + ((key ^ kl) & 15);
          kp_lds[buf][0][at] = ph;
          kp_lds[buf][1][at] = pl;
        }
      }
    };
    auto largest = [&](int slot, int from) __attribute__((always_inline)) {
      const uint4 m = *reinterpret_cast<const uint4 *>(most_lds[slot] + from);
      return __builtin_amdgcn_readfirstlane(max(max(m.x, m.y), max(m.z, m.w)));
    };
    auto smallest = [&](int slot, int from) __attribute__((always_inline)) {
      const uint4 m = *reinterpret_cast<const uint4 *>(least_lds[slot] + from);
      return __builtin_amdgcn_readfirstlane(min(min(m.x, m.y), min(m.z, m.w)));
    };

    half8 qh[G], ql[G];
    float inv_q = 0.0f;
    int row_lo = 0, wave_lo = 0;  // keys from row_lo on are seen by the row, from wave_lo on by all rows of the wave
    if (busy) {
      const TreeQuery<D> q(a.queries, a.seq[unit.b].group0 + row0 / 16 * a.Hkv + unit.h);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        qh[g] = q.piece(0, g)[lane];
        ql[g] = q.piece(1, g)[lane];
      }
      inv_q = q.inverse()[col];
      row_lo = q.from()[col];
    }
    load(t0);
    if (a.window > 0) {
      wave_lo = row_lo;
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) wave_lo = max(wave_lo, __shfl_xor(wave_lo, d));
    }

    f32x4 o[DT];
    // Weights are 2^(score - m): m is 8 below the largest score so far, or up to 15 below it;
    // not less than 8 below where the numbers there are further apart, as 2^16 is no binary16.
    float m = NEG_INF, l = 0.0f;
    bool poison = false;
    int units = 0;  // the wave's rows' unit, as a float's exponent, or -1: each its own, in unit_lds
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int tile, bool parts) __attribute__((always_inline)) {
      const int buf = tile & 1;
      const bool own = tile >= cached;
      const int base = lo + tile * BN;
      // Steps of two operands of either product, six instructions; their LDS reads run
      // AHEAD - 1 steps before them. The scores' are two 16 keys of 32 channels each,
      // the outputs' 32 keys of two 16 channels.
      constexpr int KS = G * KB / 2, VS = VB * DT / 2;
      half8 fh[AHEAD][2], fl[AHEAD][2];
      auto read = [&](int step) __attribute__((always_inline)) {
        half8 (&th)[2] = fh[step % AHEAD], (&tl)[2] = fl[step % AHEAD];
        if (step < KS) {
          const int g = step / (KB / 2), k = step % (KB / 2) * 2;
          const int at = (k * G + g) * 64 + kq * 16 + ((col ^ (4 * g + kq)) & 15);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            th[i] = kp_lds[buf][0][at + i * G * 64];
            tl[i] = kp_lds[buf][1][at + i * G * 64];
          }
        } else if (step < KS + VS) {
          const int v = (step - KS) / (DT / 2), d = (step - KS) % (DT / 2) * 2;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = (v * DT + d + i) * 64 + kq * 16 + (col ^ ((d + i) & 3));
            th[i] = vp_lds[buf][0][at];
            tl[i] = vp_lds[buf][1][at];
          }
        }
      };
      f32x4 sc[KB];
#pragma unroll
      for (int k = 0; k < KB; ++k) sc[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < AHEAD - 1; ++i) read(i);
#pragma unroll
      for (int step = 0; step < KS; ++step) {
        const int g = step / (KB / 2), k = step % (KB / 2) * 2;
        read(step + AHEAD - 1);
        __builtin_amdgcn_sched_barrier(0);
        const half8 (&th)[2] = fh[step % AHEAD], (&tl)[2] = fl[step % AHEAD];
#pragma unroll
        for (int i = 0; i < 2; ++i) sc[k + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th[i], qh[g], sc[k + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) sc[k + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th[i], ql[g], sc[k + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) sc[k + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(tl[i], qh[g], sc[k + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      // (finite and above 0: hidden scores stay -inf)
      const float f = fminf(fmaxf(inv_q * inverse_scale(kbits), 1.1754944e-38f), 3.402823466e38f);
      if (own || parts || base + BN > past || base < wave_lo) {
#pragma unroll
        for (int v = 0; v < VB; ++v) {
          const int first = 32 * v;  // of the tile
          unsigned seen;
          if (own) {
            const int w = ((tile - cached) * BN + first) / 32;
            seen = w < kMaskWords && w * 32 < nodes
                       ? a.mask[(long)(a.seq[unit.b].first + min(row0 + col, rows - 1) / a.R) * kMaskWords + w]
                       : 0u;
          } else {
            const int from = max(0, row_lo - base - first), to = min(32, past - base - first);
            seen = from >= 32 || to <= from ? 0u : (0xffffffffu << from) & (0xffffffffu >> (32 - to));
          }
          if (__builtin_expect(parts, 0)) {
            poison |= (seen & bad_lds[v]) != 0;
            seen &= take_lds[v];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(seen >> ((i & 3) + 4 * kq + 16 * (i >> 2)) & 1u)) sc[2 * v + (i >> 2)][i & 3] = NEG_INF;
        }
      }
      float big = NEG_INF;
#pragma unroll
      for (int k = 0; k < KB; ++k) big = fmaxf(big, fmaxf(fmaxf(sc[k][0], sc[k][1]), fmaxf(sc[k][2], sc[k][3])));
      big = max32(max16(big)) * f;
      if (__any(big - m > 15.0f)) {
        const float below = big - (big - (big - 8.0f) > 8.0f ? 0.0f : 8.0f);
        const float next = big - m > 15.0f ? below : m, keep = fast_exp2(m - safe_max(next));
        m = next;
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= keep;
      }
      const float off = -safe_max(m);
      int lift = 0;  // what the row's unit is above the values' scale
      const int scale = (int)(vbits >> 23);
      if (__builtin_expect(units != scale, 0)) {
        int unit = units >= 0 ? units : unit_lds[wave][col];
        float most = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) most = fmaxf(fmaxf(most, fmaxf(fabsf(o[d][0]), fabsf(o[d][1]))), fmaxf(fabsf(o[d][2]), fabsf(o[d][3])));
        most = max32(max16(most));
        const int held = (int)(__float_as_uint(most) >> 23) - 127;
        // (the largest weight of the tile is 2^weight; times the lift it stays below 2^15)
        const int weight = (int)ceilf(fmaxf(big + off, -1000.0f)), room = 15 - weight;
        int shift = scale - unit;
        if (shift > 0 && most > 0.0f) shift = min(shift, max(0, 64 - held));
        if (shift < 0 && weight < 0 && (most > 0.0f ? held + shift < 16 : weight > -1000)) shift = min(0, shift + room);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] = __builtin_ldexpf(o[d][i], shift);
        }
        unit += shift;
        unit_lds[wave][col] = unit;
        lift = unit - scale;
        const int first = __builtin_amdgcn_readfirstlane(unit);
        units = __all(unit == first) ? first : -1;
      }
      const bool lifted = units != scale;
      half8 ph[VB], pl[VB];
#pragma unroll
      for (int v = 0; v < VB; ++v) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = fast_exp2(fmaf(sc[2 * v + (i >> 2)][i & 3], f, off));
          l += p[i];
        }
        if (__builtin_expect(lifted, 0)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = __builtin_ldexpf(p[i], lift);
        }
        split8(p, minus_one, &ph[v], &pl[v]);
      }
#pragma unroll
      for (int step = KS; step < KS + VS; ++step) {
        const int v = (step - KS) / (DT / 2), d = (step - KS) % (DT / 2) * 2;
        read(step + AHEAD - 1);
        __builtin_amdgcn_sched_barrier(0);
        const half8 (&th)[2] = fh[step % AHEAD], (&tl)[2] = fl[step % AHEAD];
#pragma unroll
        for (int i = 0; i < 2; ++i) o[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th[i], ph[v], o[d + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) o[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th[i], pl[v], o[d + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) o[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(tl[i], ph[v], o[d + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    constexpr unsigned kInfinite = 0x7f800000u;
    constexpr unsigned kTop = (127u + 15u) << 23, kLow = (2u * 127u - 2u) << 23;  // 2^15; 2^-2, biased twice
    // Between two barriers a wave writes its share of a tile and computes its part of the
    // one before. A tile that has to be written again takes a turn of its own, one in
    // parts two for each but the last. In the first turn there is nothing to compute, and
    // the scales are set between reading the tile's largest and writing it.
    enum : int { kLook, kFits, kParts, kNextPart };  // (of the tile that is written: to be looked at, or why it was written again)
    int mode = kLook;
#pragma unroll 1
    for (int tile = t0 - 1; tile < t1;) {
      // (addresses anew each time)
      asm volatile("" : "+v"(thread_key), "+v"(thread_channel), "+v"(kl), "+v"(vl), "+v"(vb0), "+v"(vq), "+v"(col), "+v"(kq));
      bool again = mode == kNextPart;
      if (tile >= t0 && mode == kLook) {
        const uint2 unfit = *reinterpret_cast<const uint2 *>(unfit_lds[tile & 1]);
        again = __builtin_amdgcn_readfirstlane(unfit.x | unfit.y) != 0;
        if (__builtin_expect(again, 0)) {
          const unsigned km = largest(tile & 1, 4), vm = largest(tile & 1, 0);
          const unsigned ks = smallest(tile & 1, 4), vs = smallest(tile & 1, 0);
          mode = kFits;
          if (km >= kInfinite || vm >= kInfinite || (ks >> 23) + kSpan < km >> 23 || (vs >> 23) + kSpan < vm >> 23) {
            mode = kParts;
            for (int i = tid; i < 2 * BN; i += 512) size_lds[i] = 0;
            if (tid < VB) bad_lds[tid] = 0;
          } else {
            kbits = scale_to(unbits(km), 11);
            vbits = scale_to(unbits(vm), 11);
          }
        }
      }
      const bool hold = !again && mode == kParts && __builtin_amdgcn_readfirstlane(scale_lds[2]);  // (a part of the tile is still to be written)
      const int target = again ? tile : hold ? t1 : tile + 1;
      if (__builtin_expect(again, 0)) {
        load(tile);
        __syncthreads();  // (the tile's largest is read)
      }
      if (target < t1) {
        f32x4 cur[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cur[i] = raw[i];
        if (__builtin_expect(again && mode != kFits, 0)) {
          if (mode == kParts) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int key = thread_key + step_key(i);
              const unsigned of = bits_of(cur[i]);
              if (of >= kInfinite) atomicOr(&bad_lds[key >> 5], 1u << (key & 31));
              else atomicMax(&size_lds[(values ? BN : 0) + key], of);
            }
            __syncthreads();
          }
          if (wave == 0) {  // the next part: the largest keys left, and of those the largest values
            constexpr int PER = (BN + 63) / 64;
            unsigned key_size[PER], value_size[PER], km = 0, vm = 0;
            bool in[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int key = min(lane + 64 * i, BN - 1);
              const unsigned words = mode == kParts ? ~bad_lds[key >> 5] : left_lds[key >> 5];
              in[i] = lane + 64 * i < BN && (words >> (key & 31) & 1u);
              key_size[i] = in[i] ? size_lds[key] : 0;
              value_size[i] = size_lds[BN + key];
              km = max(km, key_size[i]);
            }
            km = wave_max_bits(km);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const bool near = in[i] && (key_size[i] == 0 || (key_size[i] >> 23) + kSpan >= km >> 23);
              value_size[i] = near ? value_size[i] : kInfinite;
              vm = max(vm, near ? value_size[i] : 0u);
            }
            vm = wave_max_bits(vm);
            bool more = false;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const bool now = value_size[i] == 0 || (value_size[i] < kInfinite && (value_size[i] >> 23) + kSpan >= vm >> 23);
              const unsigned long long taken = __ballot(now), left = __ballot(in[i] && !now);
              more |= left != 0;
              if (lane < min(2, VB - 2 * i)) {
                take_lds[2 * i + lane] = (unsigned)(taken >> (32 * lane));
                left_lds[2 * i + lane] = (unsigned)(left >> (32 * lane));
              }
            }
            if (lane == 0) {
              scale_lds[0] = scale_to(unbits(km), 11);
              scale_lds[1] = scale_to(unbits(vm), 11);
              scale_lds[2] = more;
            }
          }
          __syncthreads();
          kbits = __builtin_amdgcn_readfirstlane(scale_lds[0]);
          vbits = __builtin_amdgcn_readfirstlane(scale_lds[1]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = thread_key + step_key(i);
            if (!(take_lds[key >> 5] >> (key & 31) & 1u)) cur[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
          }
          mode = kParts;
        }
        uint2 ends;
        if (!again) ends = post(target & 1, cur);
        if (tile < t0) {
          __syncthreads();
          kbits = scale_to(unbits(min(largest(t0 & 1, 4), kInfinite - 1)), 11);
          vbits = scale_to(unbits(min(largest(t0 & 1, 0), kInfinite - 1)), 11);
          units = (int)(vbits >> 23);
        }
        if (!again && lane == 0) {  // (a number times the scale, by exponents: bits of both less the bias)
          const unsigned of = values ? vbits : kbits;
          unfit_lds[target & 1][wave] = ends.x >= kInfinite || ends.x > kTop + (127u << 23) - of || ends.y < kLow - min(of, kLow);
        }
        write(target & 1, cur);
      }
      if (target + 1 < t1) {
        load(target + 1);
      } else {  // (what the registers hold is of no use: nothing to keep across the turn)
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "=v"(raw[i]));
      }
      if (!again) {
        if (tile >= t0 && busy) compute(tile, mode == kParts);
        mode = hold ? kNextPart : kLook;
        if (!hold) ++tile;
      }
      __syncthreads();
    }

    l = sum32(sum16(l));
    if (poison) l = __builtin_nanf("");
    if (busy) {
      // (not their product: it would be below 2^-126 for the smallest values)
      const float inv = l == 0.0f ? 0.0f : 1.0f / l, down = inverse_scale((unsigned)(units >= 0 ? units : unit_lds[wave][col]) << 23);
      if (row0 + col < rows) {
        const int node = (row0 + col) / a.R;
        const long orow = (long)(a.seq[unit.b].first + node) * a.Hq + unit.h * a.R + (row0 + col - node * a.R);
        const bool whole = t0 == 0 && t1 == unit.tiles;
        float *const out = whole ? a.out + orow * D : a.part + ((long)slot_of * a.total + orow) * (D + 4);
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(out + 16 * d + 4 * kq) = o[d] * inv * down;
        if (!whole) {
          if (kq == 0) *reinterpret_cast<float2 *>(out + D) = make_float2(m, l);
        } else if (!(l > 0.0f) || l > 3.402823466e38f) {
          atomicOr(a.err, kDevErrSoftmaxDenominator);
        }
      }
    }
  }
}

// The outputs of a unit's workgroups, each divided by its own sum, by their sums'
// shares. D / 4 threads an output row and SL lanes over the workgroups, each with eight
// loads in flight. Bound by latency (3 to 5 us), with many rows by the partial outputs'
// reads (16 sequences: 8 us).
// Grid: (blocks of rows), 256 threads.
template <int D, int SL, int MB>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgsOf<MB> a) {
  constexpr int TR = D / 4, ROWS = 256 / (TR * SL), AT_ONCE = 8;
  __shared__ f32x4 acc_lds[SL > 1 ? ROWS : 1][SL][TR];
  __shared__ float2 ml_lds[SL > 1 ? ROWS : 1][SL];
  const int c = threadIdx.x % TR, sl = threadIdx.x / TR % SL, in = threadIdx.x / (TR * SL);
  const int row = blockIdx.x * ROWS + in;
  int splits = 0;
  if (row < a.total) {
    const int n = row / a.Hq, hq = row - n * a.Hq, h = hq / a.R;
    int b = 0;
    while (b < a.B - 1 && n >= a.seq[b + 1].first) ++b;
    const int block = ((n - a.seq[b].first) * a.R + (hq - h * a.R)) / a.per;
    const int start = a.seq[b].start + (block * a.Hkv + h) * a.seq[b].padded;
    splits = (start + a.seq[b].tiles - 1) / a.share - start / a.share + 1;
  }
  if (splits == 1) splits = 0;  // (its workgroup has written the output)
  float m = NEG_INF, l = 0.0f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i = sl; i < splits; i += SL * AT_ONCE) {
    float2 ml[AT_ONCE];
    f32x4 x[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const float *const part = a.part + ((long)min(i + j * SL, splits - 1) * a.total + row) * (D + 4);
      ml[j] = *reinterpret_cast<const float2 *>(part + D);
      x[j] = reinterpret_cast<const f32x4 *>(part)[c];
    }
    float big = m;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (i + j * SL >= splits) ml[j] = make_float2(NEG_INF, 0.0f);
      big = fmaxf(big, ml[j].x);
    }
    const float keep = fast_exp2(m - safe_max(big));
    l *= keep;
    acc *= keep;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const float w = ml[j].y * fast_exp2(ml[j].x - safe_max(big));
      l += w;
      acc += x[j] * w;
    }
    m = big;
  }
  if constexpr (SL > 1) {
    acc_lds[in][sl][c] = acc;
    if (c == 0) ml_lds[in][sl] = make_float2(m, l);
    __syncthreads();
    if (sl != 0) return;
#pragma unroll
    for (int i = 1; i < SL; ++i) m = fmaxf(m, ml_lds[in][i].x);
    l = 0.0f;
    acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const float w = fast_exp2(ml_lds[in][i].x - safe_max(m));
      l = fmaf(ml_lds[in][i].y, w, l);
      acc += acc_lds[in][i][c] * w;
    }
  }
  if (splits == 0) return;
  if (c == 0 && (!(l > 0.0f) || l > 3.402823466e38f)) atomicOr(a.err, kDevErrSoftmaxDenominator);
  reinterpret_cast<f32x4 *>(a.out + (long)row * D)[c] = acc * (1.0f / l);
}

// A workgroup's share of the tiles: a cus'th of them all. Units start with a
// workgroup of their own, their tiles padded to whole shares, where that takes shares
// at most an eighth larger (26 nodes over 8192 rows: 32.4 us against 35.1 end to end, 256
// over 32768: 135.5 against 145); else they lie end to end, and a workgroup at a border
// takes both sides (a start more). False where there are more places than an int has.
bool tree_plan(int D, int R, int Hkv, int window, const int *past, const int *nodes, int B, int cus, TreePlan *plan) {
  const int BN = 8192 / D;
  TreePlan &p = *plan;
  p = TreePlan{};
  const int per = kTreeRows;
  long units[kMaxDecodeBatch], total = 0;
  for (int b = 0; b < B; ++b) {
    const int lo = window > 0 ? std::max(0, past[b] + 1 - window) : 0;
    p.tiles[b] = nodes[b] ? (past[b] - lo + BN - 1) / BN + (nodes[b] + BN - 1) / BN : 1;
    units[b] = (long)((nodes[b] * (long)R + per - 1) / per) * Hkv;
    total += units[b] * p.tiles[b];
    p.group0[b] = p.groups;
    p.groups += ((long)nodes[b] * R + 15) / 16 * Hkv;
  }
  // (two tiles: a turn more costs less than the merge, 4 sequences of 16 nodes over 125 keys
  // of 8 heads of 64 13.7 us against 14.1, over 29 of 256 15.8 against 18.3; three: 16.1
  // against 14.6 and 17.9 against 19.9, and one sequence 2 us the other way)
  const int longest = *std::max_element(p.tiles, p.tiles + B);
  const long least = std::max<long>(longest <= 2 ? 2 : 1, (total + cus - 1) / cus);
  if (total > (1 << 30) || least > (1 << 30)) return false;
  bool padded = false;
  long share = least;
  for (; share <= least + least / 8 + 1; ++share) {
    long groups = 0;
    for (int b = 0; b < B; ++b) groups += units[b] * ((p.tiles[b] + share - 1) / share);
    padded = groups <= cus;
    if (padded) break;
  }
  p.share = (int)(padded ? share : least);
  for (int b = 0; b < B; ++b) {
    const int shares = (p.tiles[b] + p.share - 1) / p.share;
    p.padded[b] = padded ? shares * p.share : p.tiles[b];
    p.start[b] = p.places;
    p.places += (int)(units[b] * p.padded[b]);
    // (end to end, a unit may begin and end within others' workgroups)
    if (nodes[b]) p.splits = std::max(p.splits, padded ? shares : (p.tiles[b] + p.share - 2) / p.share + 1);
  }
  return true;
}

template <int D, int MB>
static void run_merge(hipStream_t st, const TreeArgsOf<MB> &a, int splits) {
  constexpr int TR = D / 4;
  auto run = [&](auto lanes) {
    constexpr int SL = decltype(lanes)::value, ROWS = 256 / (TR * SL);
    hipLaunchKernelGGL((tree_merge_kernel<D, SL, MB>), dim3((a.total + ROWS - 1) / ROWS), dim3(256), 0, st, a);
  };
  // (a step with 26 or 33 workgroups a unit: 34.0 and 24.5 us with one lane a row, 32.8 and
  // 22.8 with four; 16 sequences, 9 or fewer: 145.9 with one, 146.8 with four)
  if (splits <= 8) run(std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, 4>{});
}

template <int D, int MB>
static void run_attend(hipStream_t st, const TreeArgsOf<MB> &a, const TreePlan &p) {
  int lines = 0;  // of the prepare kernel: queries, keys and values
  for (int b = 0; b < a.B; ++b) {
    const int n = a.seq[b].nodes;
    lines = std::max(lines, (((n * a.R + 15) & ~15) + 2 * n) * a.Hkv);
  }
  constexpr int LINES = 2048 / D;
  hipLaunchKernelGGL((tree_prepare_kernel<D, MB>), dim3((lines + LINES - 1) / LINES, a.B), dim3(256), 0, st, a);
  hipLaunchKernelGGL((tree_attend_kernel<D, MB>), dim3((a.places + a.share - 1) / a.share), dim3(512), 0, st, a);
  if (p.splits > 1) run_merge<D>(st, a, p.splits);
}

template <int MB>
static hipError_t run_tree(hipStream_t st, const TreeArgsOf<MB> &a, const TreePlan &p, int D) {
  if (D == 64) run_attend<64>(st, a, p);
  else if (D == 128) run_attend<128>(st, a, p);
  else run_attend<256>(st, a, p);
  return hipGetLastError();
}

hipError_t launch_tree(hipStream_t st, TreeArgs &a, const TreePlan &p, int D) {
  a.share = p.share;
  a.places = p.places;
  a.per = kTreeRows;
  for (int b = 0; b < a.B; ++b) {
    a.seq[b].start = p.start[b];
    a.seq[b].tiles = p.tiles[b];
    a.seq[b].padded = p.padded[b];
    a.seq[b].group0 = p.group0[b];
  }
  if (a.B > 1) return run_tree(st, a, p, D);
  TreeArgsOf<1> one;  // (a launch's arguments cost time: 16.2 us a step of five nodes, 17.2 with room for 16 sequences)
  static_cast<TreeBase &>(one) = a;
  one.seq[0] = a.seq[0];
  return run_tree(st, one, p, D);
}

// The walk along confirmed nodes: every node that holds the token sampled at its
// parent offers itself as the parent's next, the lowest one stays, and one thread
// follows them. Bound by latency: a load, an LDS read a node of the path, a store (5 nodes
// 1.8 us, 64 trees of up to 64 nodes 3 us).
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
// latency: the path, then one round of loads and one of stores (28 caches, 4 rows of 8 x
// 128: 3.6 us; 32 caches, 12 rows: 5.2 us).
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
