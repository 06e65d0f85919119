// tree.hip -- decoding with drafted tokens: a tree of them through one layer's
// attention, the walk along those that sampling confirms, and the move of their
// rows in the caches.
//
// The step. Node t of a sequence of P cached rows has the position P + depth(t)
// and sees the cached rows (with a window those less than W positions before it),
// the nodes it descends from and itself. Its key, rotated at its position, and its
// value become the cache's row P + t, and
//   out_t = sum_j p_tj v_j,  p_t = softmax_j(q_t . k_j / sqrt(d)).
#include <type_traits>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

constexpr int kMaskWords = kTreeMaxNodes / 32;

// Each thread's node (of up to 256): its depth and, with MASKS, the nodes that it
// sees, by doubling: after k rounds a node knows the 2^k nodes above it. A parent
// out of its range counts as none. For 256 threads.
struct TreeShape {
  int depth[kTreeMaxNodes];
  int above[kTreeMaxNodes];  // the node 2^k above
  unsigned mask[kTreeMaxNodes][kMaskWords];
};
template <bool MASKS>
__device__ void tree_shape(const int *parents, int nodes, TreeShape &s, int *err) {
  const int t = threadIdx.x;
  int p = t < nodes ? parents[t] : -1;
  if (p < -1 || p >= t) {
    if (err) atomicOr(err, kDevErrTreeParent);
    p = -1;
  }
  int depth = p >= 0 ? 1 : 0;
  unsigned m[kMaskWords] = {};
  if constexpr (MASKS) {
#pragma unroll
    for (int w = 0; w < kMaskWords; ++w) m[w] = t >> 5 == w ? 1u << (t & 31) : 0u;
  }
  for (int span = 1;; span *= 2) {
    s.depth[t] = depth;
    s.above[t] = p;
    if constexpr (MASKS) {
#pragma unroll
      for (int w = 0; w < kMaskWords; ++w) s.mask[t][w] = m[w];
    }
    __syncthreads();
    if (span >= nodes) return;
    int up = -1;
    if (p >= 0) {
      depth += s.depth[p];
      up = s.above[p];
      if constexpr (MASKS) {
#pragma unroll
        for (int w = 0; w < kMaskWords; ++w) m[w] |= s.mask[p][w];
      }
    }
    p = up;
    __syncthreads();
  }
}

}  // namespace

// Queries, keys and values of the nodes: the norm, the rotation at the node's
// position, the rows into the cache (and its bf16 operands). D / 8 threads a row,
// each with four channels and their rotation's partners, half a row on.
// Grid: (row blocks of the longest sequence, sequences), 256 threads.
template <int D>
__global__ __launch_bounds__(256) void tree_prepare_kernel(const TreeArgs a) {
  __shared__ TreeShape shape;
  constexpr int TR = D / 8, ROWS = 256 / TR;
  const TreeSeq &s = a.seq[blockIdx.y];
  const int per = a.Hq + 2 * a.Hkv, total = s.nodes * per;
  if ((int)blockIdx.x * ROWS >= total) return;
  if (blockIdx.x == 0) {
    tree_shape<true>(a.parents + s.first, s.nodes, shape, a.err);
    const int t = threadIdx.x;
    if (t < s.nodes) {
      a.depth[s.first + t] = shape.depth[t];
#pragma unroll
      for (int w = 0; w < kMaskWords; ++w) a.mask[(long)(s.first + t) * kMaskWords + w] = shape.mask[t][w];
    }
  } else {
    tree_shape<false>(a.parents + s.first, s.nodes, shape, nullptr);
  }
  const int row = blockIdx.x * ROWS + threadIdx.x / TR, c = threadIdx.x % TR * 4;
  if (row >= total) return;
  const int node = row / per, hh = row - node * per;
  const int kind = hh < a.Hq ? 0 : hh < a.Hq + a.Hkv ? 1 : 2;
  const int h = kind == 0 ? hh : kind == 1 ? hh - a.Hq : hh - a.Hq - a.Hkv;
  const float *src = kind == 0 ? a.q + ((long)(s.first + node) * a.Hq + h) * D
                               : (kind == 1 ? a.k : a.v) + ((long)(s.first + node) * a.Hkv + h) * D;
  const float4 x = *reinterpret_cast<const float4 *>(src + c), y = *reinterpret_cast<const float4 *>(src + D / 2 + c);
  float lo[4] = {x.x, x.y, x.z, x.w}, hi[4] = {y.x, y.y, y.z, y.w};
  const long at = s.past + node;
  if (kind < 2) {
    if (a.q_norm) {
#pragma clang fp contract(off)
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += lo[i] * lo[i] + hi[i] * hi[i];
      const float inv = 1.0f / sqrtf(group_sum<TR>(sum) / (float)D + a.eps);
      const float *w = kind == 0 ? a.q_norm : a.k_norm;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = lo[i] * inv * w[c + i];
        hi[i] = hi[i] * inv * w[D / 2 + c + i];
      }
    }
    if (a.cos) {
      const long pos = (s.past + shape.depth[node]) * (long)(D / 2) + c;
#pragma unroll
      for (int i = 0; i < 4; ++i) rotate_pair(lo[i], hi[i], a.cos[pos + i], a.sin[pos + i]);
    }
  }
  float *dst;
  if (kind == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] *= a.prescale;
      hi[i] *= a.prescale;
    }
    dst = a.q_rot + ((long)(s.first + node) * a.Hq + h) * D;
  } else {
    dst = (kind == 1 ? s.k : s.v) + (at * a.Hkv + h) * D;
  }
  *reinterpret_cast<float4 *>(dst + c) = make_float4(lo[0], lo[1], lo[2], lo[3]);
  *reinterpret_cast<float4 *>(dst + D / 2 + c) = make_float4(hi[0], hi[1], hi[2], hi[3]);
  if (kind == 1 && s.kb) {
    bf16 *kb = s.kb + ((long)h * s.cap + at) * D + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kb[i] = (bf16)lo[i];
      kb[D / 2 + i] = (bf16)hi[i];
    }
  } else if (kind == 2 && s.kb) {
    bf16 *vt = s.vt + ((long)h * D + c) * s.cap + vt_key_slot(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vt[i * s.cap] = (bf16)lo[i];
      vt[(D / 2 + i) * s.cap] = (bf16)hi[i];
    }
  }
}

// Attention of one node and query head a wave, key by key.
// Grid: (nodes of the longest sequence, ceil(Hq / 4), sequences), 256 threads.
template <int D>
__global__ __launch_bounds__(256) void tree_attend_kernel(const TreeArgs a) {
  constexpr int E = D / 64;
  const TreeSeq &s = a.seq[blockIdx.z];
  const int node = blockIdx.x, hq = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (node >= s.nodes || hq >= a.Hq) return;
  const int h = hq / a.R, depth = a.depth[s.first + node], pos = s.past + depth;
  const unsigned *mask = a.mask + (long)(s.first + node) * kMaskWords;
  const long orow = ((long)(s.first + node) * a.Hq + hq) * D + lane * E;
  float q[E], o[E], m = NEG_INF, l = 0.0f;
  bool wrong = false;  // a key or value that is not finite
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = a.q_rot[orow + e] * a.qscale;
    o[e] = 0.0f;
  }
  auto key = [&](int j) {
    const long at = ((long)j * a.Hkv + h) * D + lane * E;
    float dot = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float k = s.k[at + e], v = s.v[at + e];
      wrong |= !(fabsf(k) < __builtin_inff()) || !(fabsf(v) < __builtin_inff());
      dot = fmaf(q[e], k, dot);
    }
    const float x = group_sum<64>(dot), big = fmaxf(m, x);
    const float keep = fast_exp2(m - safe_max(big)), p = fast_exp2(x - safe_max(big));
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], keep, p * s.v[at + e]);
    m = big;
  };
  for (int j = a.window > 0 ? max(0, pos + 1 - a.window) : 0; j < s.past; ++j) key(j);
  for (int t = 0; t <= node; ++t)
    if (mask[t >> 5] >> (t & 31) & 1u && (a.window <= 0 || depth - a.depth[s.first + t] < a.window)) key(s.past + t);
  if (__any(wrong)) l = __builtin_nanf("");
  if (!(l > 0.0f) || l > 3.402823466e38f) {
    if (lane == 0) atomicOr(a.err, kDevErrSoftmaxDenominator);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) a.out[orow + e] = o[e] / l;
}

hipError_t launch_tree(hipStream_t st, const TreeArgs &a, int D, int B) {
  int most = 0;
  for (int b = 0; b < B; ++b) most = a.seq[b].nodes > most ? a.seq[b].nodes : most;
  const int rows = 256 / (D / 8);
  const dim3 prepare((unsigned)((most * (long)(a.Hq + 2 * a.Hkv) + rows - 1) / rows), B);
  const dim3 attend(most, (a.Hq + 3) / 4, B);
  auto run = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    hipLaunchKernelGGL(tree_prepare_kernel<DD>, prepare, dim3(256), 0, st, a);
    hipLaunchKernelGGL(tree_attend_kernel<DD>, attend, dim3(256), 0, st, a);
  };
  if (D == 64) run(std::integral_constant<int, 64>{});
  else if (D == 128) run(std::integral_constant<int, 128>{});
  else run(std::integral_constant<int, 256>{});
  return hipGetLastError();
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
  const int t = threadIdx.x;
  int count = a.count[c.seq];
  bool wrong = count < 0 || count > c.nodes;
  count = min(max(count, 0), c.nodes);
  if (t == 0) end = count;
  __syncthreads();
  if (t < count) {
    const int p = a.path[c.first + t];
    path[t] = p;
    if (p < 0 || p >= c.nodes || (t > 0 && p <= a.path[c.first + t - 1])) {
      wrong = true;
      atomicMin(&end, t);
    }
  }
  if (wrong && blockIdx.x == 0 && !values) atomicOr(a.err, kDevErrTreePath);
  __syncthreads();
  const int n = end;
  const long width = (long)c.heads * c.dim, P = c.past;
  const long unit = (long)blockIdx.x * 256 + t;
  char *const rows = values ? c.v : c.k;
  if (c.kind == 2) {
    // pieces of a head's codes, then its words of step and minimum
    const int pieces = c.dim / 32, words = c.dim / 32;
    const long h = unit / (pieces + words);
    const int i = (int)(unit - h * (pieces + words));
    if (h >= c.heads) return;
    if (i < pieces) {
      char *const p = rows + (h * c.cap + P) * (c.dim / 2) + i * 16;
      move_rows<uint4>(path, n, [&](int r) { return p + (long)r * (c.dim / 2); });
    } else {
      char *const p = (values ? c.vp : c.kp) + ((h * c.cap + P) * words + (i - pieces)) * 4;
      move_rows<unsigned>(path, n, [&](int r) { return p + (long)r * words * 4; });
    }
    return;
  }
  const bool wide = width % 4 == 0;
  if (unit < (wide ? width / 4 : width)) {
    char *const p = rows + (P * width + unit * (wide ? 4 : 1)) * 4;
    if (wide) move_rows<uint4>(path, n, [&](int r) { return p + (long)r * width * 4; });
    else move_rows<unsigned>(path, n, [&](int r) { return p + (long)r * width * 4; });
  }
  if (c.kind == 0) return;
  if (!values) {  // bf16 keys [H, cap, D], eight a thread
    const long h = unit / (c.dim / 8);
    const int i = (int)(unit - h * (c.dim / 8));
    if (h >= c.heads) return;
    char *const p = c.kp + ((h * c.cap + P) * c.dim + i * 8) * 2;
    move_rows<uint4>(path, n, [&](int r) { return p + (long)r * c.dim * 2; });
  } else {  // bf16 values [H, D, cap], four channels a thread
    for (long i = unit * 4; i < min(unit * 4 + 4, width); ++i) {
      char *const p = c.vp + i * c.cap * 2;
      move_rows<unsigned short>(path, n, [&](int r) { return p + vt_key_slot(P + r) * 2; });
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
