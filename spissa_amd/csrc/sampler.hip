// sampler.hip -- one token of each row of logits: temperature, top-k, top-p and
// min-p, and a given random number.
//
// All three filters keep the first tokens in the order of falling logits (equal ones
// by index), so what is kept is known by its last token. Weights w = exp((x - max) / T)
// are formed in 64 bits and held as whole numbers of 2^-shift: their sums are exact,
// whatever the order, and the limits are met where the definition has them (sums in
// single precision would move the borders of some hundred thousand tokens by 2^-24, and
// one row in a hundred would come out another token).
//
// A row's logits are read three times, by workgroups of a slice each:
//   1. the slice's largest and smallest logit;
//   2. counts and weights of 1024 bins of (max - x), fine enough that few tokens share
//      the bin in which a filter ends;
//   3. with those bins known: their tokens into a list, and the sum of the weights
//      certain to be kept.
// Between and after them a workgroup a row finds the bins, then sorts the list (of some
// hundred tokens), finds the last kept one, draws, and walks the slice in which the draw
// falls. A row whose list would not fit (thousands of tokens within a thousandth of the
// logits' range) is done by bits of the logits instead, by a workgroup over the whole
// row. Bound by latency for a few rows; for many by the reads and by the weights' 30
// operations in 64 bits a token.
#include <algorithm>
#include <climits>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

typedef unsigned long long u64;

constexpr int NT = 512, BINS = 1024, LIST = 4096;

// Bits that rise with the value; both zeros alike.
__device__ __forceinline__ unsigned sort_key(float x) {
  const unsigned b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

// exp((x - max) / T) as 2^(n + r), |r| <= 1/2, by twelve terms of exp(r ln 2): off by at
// most 2^-52 of itself.
struct Weigh {
  double top, inv, min_p;  // inv: log2(e) / T
  int shift;
  __device__ __forceinline__ double real(float x, int add) const {
    const double y = fmax(((double)x - top) * inv, -1000.0);
    const double n = rint(y), r = (y - n) * 0.69314718055994530942;
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n + add);
  }
  // The nearest whole number of 2^-shift (below 2^52: the sum's low bits are it).
  __device__ __forceinline__ u64 operator()(float x) const {
    return (u64)__double_as_longlong(real(x, shift) + 4503599627370496.0) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 least(float x) const {  // 0 below min_p
    const double w = real(x, shift);
    return w >= min_p ? (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull : 0;
  }
};

// A slice's largest logit with its first place, its smallest, and whether one is NaN or +infinite.
struct Slice {
  float most, least;
  int at, bad;
};
// What a row's later passes go by.
struct Row {
  u64 whole;            // weights of all
  float top, per_bin;
  float temperature, top_p, min_p, u;
  int top_k;            // 0: all
  int state;            // kBad.. below
  int lo, hi, k;        // bins of the list: lo..hi (where top-p may end) and k (where top-k ends); certain below lo
  int need_k;           // tokens of bin k that top-k keeps
  int first;            // the largest logit's first place
  u64 before_lo, before_k;  // weights of the bins before lo and before k
};
enum : int { kBad, kGreedy, kAll, kList };

// u and the settings of a row, and whether they are in range.
__device__ __forceinline__ bool settings(const SampleArgs &a, int row, Row &r) {
  r.temperature = a.d_temperature ? a.d_temperature[row] : a.temperature;
  r.top_p = a.d_top_p ? a.d_top_p[row] : a.top_p;
  r.min_p = a.d_min_p ? a.d_min_p[row] : a.min_p;
  const int k = a.d_top_k ? a.d_top_k[row] : a.top_k;
  r.top_k = k > 0 && k < a.vocab ? k : 0;
  r.u = a.u[row];
  return r.u >= 0.0f && r.u < 1.0f && r.temperature >= 0.0f && r.temperature < __builtin_inff() && r.top_p >= 0.0f &&
         r.top_p <= 1.0f && r.min_p >= 0.0f && r.min_p <= 1.0f;
}

__device__ __forceinline__ Weigh weigh_of(const Row &r, int shift) {
  return Weigh{(double)r.top, 1.4426950408889634074 / (double)r.temperature, ldexp((double)r.min_p, shift), shift};
}

// Falls with the logit. Beyond 40 temperatures, where bins end, weights are 0.
__device__ __forceinline__ int bin_of(float x, float top, float per_bin) {
  const float t = (top - x) * per_bin;
  return t < BINS - 1 ? (int)t : BINS - 1;
}

// f(index, logit) for a thread's logits of a slice, four in a row at a time.
template <class F>
__device__ __forceinline__ void each(const float *x, int from, int to, bool vec, F f) {
  if (vec) {
    for (int i = from + 4 * (int)threadIdx.x; i < to; i += 4 * NT) {
      if (i + 4 <= to) {
        const float4 v = *reinterpret_cast<const float4 *>(x + i);
        f(i, v.x);
        f(i + 1, v.y);
        f(i + 2, v.z);
        f(i + 3, v.w);
      } else {
        for (int j = i; j < to; ++j) f(j, x[j]);
      }
    }
  } else {
    for (int i = from + (int)threadIdx.x; i < to; i += NT) f(i, x[i]);
  }
}

template <class T>
__device__ T block_sum(T v, T *part) {
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  T r = 0;
  for (int i = 0; i < NT / 64; ++i) r += part[i];
  return r;
}

// The sum of the threads' values before this one's, and of all.
template <class T>
__device__ T block_before(T v, T *part, T *all) {
  const int lane = threadIdx.x & 63;
  T run = v;
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  __syncthreads();
  if (lane == 63) part[threadIdx.x >> 6] = run;
  __syncthreads();
  T before = 0, total = 0;
  for (int i = 0; i < NT / 64; ++i) {
    if (i < (int)(threadIdx.x >> 6)) before += part[i];
    total += part[i];
  }
  *all = total;
  return before + run - v;
}

// A row's share of the workspace.
struct Space {
  Row *row;
  Slice *slices;
  u64 *kept;        // [slices]: weights certain to be kept
  u64 *weights;     // [slices][BINS]
  unsigned *counts; // [slices][BINS]
  unsigned *listed; // tokens of the list (beyond LIST: not all of them there)
  u64 *list;        // [LIST]: key, and the index's complement
};
__host__ __device__ inline size_t row_bytes(int slices) {
  return ((sizeof(Row) + 15) & ~(size_t)15) + (size_t)slices * (sizeof(Slice) + 16 + BINS * 12) + 16 + LIST * 8;
}
__device__ __forceinline__ Space space_of(char *workspace, int row, int slices) {
  char *p = workspace + (size_t)row * row_bytes(slices);
  Space s;
  s.row = reinterpret_cast<Row *>(p);
  p += (sizeof(Row) + 15) & ~(size_t)15;
  s.listed = reinterpret_cast<unsigned *>(p);
  p += 16;
  s.list = reinterpret_cast<u64 *>(p);
  p += LIST * 8;
  s.weights = reinterpret_cast<u64 *>(p);
  p += (size_t)slices * BINS * 8;
  s.kept = reinterpret_cast<u64 *>(p);
  p += (size_t)slices * 16;
  s.slices = reinterpret_cast<Slice *>(p);
  p += (size_t)slices * sizeof(Slice);
  s.counts = reinterpret_cast<unsigned *>(p);
  return s;
}

}  // namespace

struct SampleWork {
  char *space;
  int slices, length;  // of a row; logits of a slice
  int shift;
};

// Grid: (slices, rows).
__global__ __launch_bounds__(NT) void sample_ends_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ Slice part[NT / 64];
  const int row = blockIdx.y, from = blockIdx.x * w.length, to = min(a.vocab, from + w.length);
  const float *const x = a.x + (long)row * a.vocab;
  Slice s{NEG_INF, __builtin_inff(), INT_MAX, 0};
  each(x, from, to, (reinterpret_cast<uintptr_t>(x) & 15) == 0, [&](int i, float v) {
    s.bad |= !(v < __builtin_inff());
    if (v > s.most) {
      s.most = v;
      s.at = i;
    }
    s.least = fminf(s.least, v);
  });
  auto join = [&](float most, float least, int at, int bad) {
    if (most > s.most || (most == s.most && at < s.at)) s.at = at;
    s.most = fmaxf(s.most, most);
    s.least = fminf(s.least, least);
    s.bad |= bad;
  };
  for (int d = 32; d > 0; d >>= 1) join(__shfl_xor(s.most, d), __shfl_xor(s.least, d), __shfl_xor(s.at, d), __shfl_xor(s.bad, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NT / 64; ++i) join(part[i].most, part[i].least, part[i].at, part[i].bad);
    space_of(w.space, row, w.slices).slices[blockIdx.x] = s;
  }
}

// A row's ends from its slices', its settings, and what is to be done; every thread gets it.
__device__ __forceinline__ Row row_of(const SampleArgs &a, const SampleWork &w, const Space &s, int row, int *first) {
  __shared__ Slice part[NT / 64];
  Slice e{NEG_INF, __builtin_inff(), INT_MAX, 0};
  auto join = [&](float most, float least, int at, int bad) {
    if (most > e.most || (most == e.most && at < e.at)) e.at = at;
    e.most = fmaxf(e.most, most);
    e.least = fminf(e.least, least);
    e.bad |= bad;
  };
  for (int i = threadIdx.x; i < w.slices; i += NT) join(s.slices[i].most, s.slices[i].least, s.slices[i].at, s.slices[i].bad);
  for (int d = 32; d > 0; d >>= 1) join(__shfl_xor(e.most, d), __shfl_xor(e.least, d), __shfl_xor(e.at, d), __shfl_xor(e.bad, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = e;
  __syncthreads();
  for (int i = 0; i < NT / 64; ++i) join(part[i].most, part[i].least, part[i].at, part[i].bad);
  Row r;
  const bool fine = settings(a, row, r);
  r.top = e.most;
  // (bins over the logits' range, or as far as weights are above 0)
  const float range = fminf(e.most - e.least, 40.0f * r.temperature);
  r.per_bin = range > 0.0f ? fminf((BINS - 1) / range, 1e38f) : 1.0f;
  r.state = e.bad || e.most == NEG_INF || !fine ? kBad
            : r.temperature == 0.0f             ? kGreedy
            : r.top_k == 0 && r.top_p >= 1.0f   ? kAll
                                                : kList;
  *first = e.at;
  return r;
}

// Counts (for top-k) and weights (for top-p) of the slice's bins; without either filter
// the sum of its kept weights. Grid: (slices, rows).
__global__ __launch_bounds__(NT) void sample_bins_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ u64 weights[BINS], part[NT / 64];
  __shared__ unsigned counts[BINS];
  const int row = blockIdx.y, from = blockIdx.x * w.length, to = min(a.vocab, from + w.length);
  const float *const x = a.x + (long)row * a.vocab;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const Space s = space_of(w.space, row, w.slices);
  int first;
  const Row r = row_of(a, w, s, row, &first);
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.listed = 0;
  if (r.state < kAll) return;
  const Weigh weigh = weigh_of(r, w.shift);
  if (r.state == kAll) {
    u64 sum = 0;
    each(x, from, to, vec, [&](int, float v) { sum += weigh.least(v); });
    sum = block_sum(sum, part);
    if (threadIdx.x == 0) s.kept[blockIdx.x] = sum;
    return;
  }
  for (int i = threadIdx.x; i < BINS; i += NT) {
    weights[i] = 0;
    counts[i] = 0;
  }
  __syncthreads();
  const bool by_weight = r.top_p < 1.0f, by_count = r.top_k > 0;
  each(x, from, to, vec, [&](int, float v) {
    const int b = bin_of(v, r.top, r.per_bin);
    if (by_count) atomicAdd(&counts[b], 1u);
    if (by_weight && b < BINS - 1) atomicAdd(&weights[b], weigh(v));
    else if (by_weight) {
      const u64 p = weigh(v);
      if (p) atomicAdd(&weights[b], p);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) {
    if (by_weight) s.weights[(long)blockIdx.x * BINS + i] = weights[i];
    if (by_count) s.counts[(long)blockIdx.x * BINS + i] = counts[i];
  }
}

// The bins in which the filters end. Grid: rows.
__global__ __launch_bounds__(NT) void sample_cut_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ u64 part[NT / 64], before[BINS + 1];
  __shared__ unsigned parts[NT / 64];
  __shared__ int found[3];
  __shared__ unsigned above_k;
  const int row = blockIdx.x, t = threadIdx.x;
  const Space s = space_of(w.space, row, w.slices);
  int first;
  Row r = row_of(a, w, s, row, &first);
  constexpr int PER = BINS / NT;
  if (r.state == kList) {
    const bool by_weight = r.top_p < 1.0f, by_count = r.top_k > 0;
    if (t < 3) found[t] = BINS - 1;
    if (t == 0) above_k = 0;
    u64 wt[PER] = {}, run = 0, total;
    unsigned ct[PER] = {}, runs = 0, counted;
    static_assert(PER == 2, "a thread's bins are one load");
    if (by_weight) {
#pragma unroll 16
      for (int i = 0; i < w.slices; ++i) {
        const ulonglong2 v = reinterpret_cast<const ulonglong2 *>(s.weights + (long)i * BINS)[t];
        wt[0] += v.x;
        wt[1] += v.y;
      }
    }
    if (by_count) {
#pragma unroll 16
      for (int i = 0; i < w.slices; ++i) {
        const uint2 v = reinterpret_cast<const uint2 *>(s.counts + (long)i * BINS)[t];
        ct[0] += v.x;
        ct[1] += v.y;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      run += wt[j];
      runs += ct[j];
    }
    u64 up = block_before(run, part, &total);
    unsigned ups = block_before(runs, parts, &counted);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      before[t * PER + j] = up;
      up += wt[j];
      if (by_count && ups < (unsigned)r.top_k && ups + ct[j] >= (unsigned)r.top_k) {
        found[2] = t * PER + j;
        above_k = ups;
      }
      ups += ct[j];
    }
    if (t == NT - 1) before[BINS] = total;
    __syncthreads();
    int k = by_count ? found[2] : BINS;
    // (the last bin of a range cut at 40 temperatures holds no weight: nothing to tell apart)
    const bool cut_off = r.per_bin * (40.0f * r.temperature) <= BINS;
    if (k == BINS - 1 && cut_off) k = BINS;
    r.k = k;
    r.need_k = k < BINS ? r.top_k - (int)above_k : 0;
    r.before_k = k < BINS ? before[k] : 0;
    r.whole = total;
    r.lo = k;
    r.hi = k;
    if (by_weight) {
      // the sum that top-p is of lies between those without and with all of bin k
      const double least = (double)r.top_p * (double)before[k], most = (double)r.top_p * (double)before[k < BINS ? k + 1 : BINS];
      const u64 want_lo = max((u64)1, (u64)__double2ll_ru(least)), want_hi = max((u64)1, (u64)__double2ll_ru(most));
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int b = t * PER + j;
        if (before[b] < want_lo && before[b + 1] >= want_lo) found[0] = b;
        if (before[b] < want_hi && before[b + 1] >= want_hi) found[1] = b;
      }
      __syncthreads();
      r.lo = min(found[0], k);
      r.hi = min(found[1], k);
      r.before_lo = before[min(r.lo, BINS)];
    }
    if (k == BINS && !by_weight) r.state = kAll;  // (top-k takes all that has weight: its sums come in the next pass)
  }
  if (t == 0) {
    r.first = first;
    *s.row = r;
  }
}

// The tokens of the bins in which the filters end, and the sum of the certain ones.
// Grid: (slices, rows).
__global__ __launch_bounds__(NT) void sample_list_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ u64 part[NT / 64], list[LIST];
  __shared__ unsigned listed, place;
  const int row = blockIdx.y, from = blockIdx.x * w.length, to = min(a.vocab, from + w.length);
  const float *const x = a.x + (long)row * a.vocab;
  const Space s = space_of(w.space, row, w.slices);
  const Row r = *s.row;
  if (r.state < kAll || (r.state == kAll && r.top_k == 0)) return;
  const Weigh weigh = weigh_of(r, w.shift);
  const int lo = r.state == kAll ? BINS : r.lo;
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  u64 sum = 0;
  each(x, from, to, (reinterpret_cast<uintptr_t>(x) & 15) == 0, [&](int i, float v) {
    const int b = bin_of(v, r.top, r.per_bin);
    if (b < lo) {
      sum += weigh.least(v);
    } else if (b <= r.hi || b == r.k) {
      const unsigned at = atomicAdd(&listed, 1u);
      if (at < LIST) list[at] = (u64)sort_key(v) << 32 | ~(unsigned)i;
    }
  });
  sum = block_sum(sum, part);
  if (threadIdx.x == 0) {
    s.kept[blockIdx.x] = sum;
    place = listed ? atomicAdd(s.listed, listed) : 0;
  }
  __syncthreads();
  for (unsigned i = threadIdx.x; i < min(listed, (unsigned)LIST); i += NT)
    if (place + i < LIST) s.list[place + i] = list[i];
}

// The last kept token from the list, the draw, and the token. Grid: rows.
__global__ __launch_bounds__(NT) void sample_draw_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ __attribute__((aligned(16))) u64 list[LIST];
  __shared__ u64 part[NT / 64], hist[256];
  __shared__ unsigned found;
  __shared__ u64 above;
  __shared__ u64 ends[2];
  const int row = blockIdx.x, t = threadIdx.x, n = a.vocab;
  const float *const x = a.x + (long)row * n;
  const Space s = space_of(w.space, row, w.slices);
  const Row r = *s.row;
  auto answer = [&](int token, float prob) {
    a.tokens[row] = token;
    if (a.probs) a.probs[row] = prob;
  };
  if (r.state == kBad || r.state == kGreedy) {
    if (t == 0) {
      if (r.state == kBad) atomicOr(a.err, kDevErrSampling);
      r.state == kBad ? answer(-1, 0.0f) : answer(r.first, 1.0f);
    }
    return;
  }
  const Weigh weigh = weigh_of(r, w.shift);
  unsigned last = 0;        // the last kept token's key,
  unsigned last_at = UINT_MAX;  // and index: none of that key after it is kept
  const unsigned listed = r.state == kList ? *s.listed : 0;
  if (listed > LIST) {
    // Eight bits of the keys a round, the highest first: the key at which the running
    // sum from above (of `value` over keys above `floor`) reaches `want`, and what is above it.
    auto select = [&](auto value, u64 want, unsigned floor, bool all, u64 *over) {
      unsigned prefix = 0;
      u64 sum = 0;
      for (int at = 24; at >= 0; at -= 8) {
        __syncthreads();
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int i = t; i < n; i += NT) {
          const unsigned k = sort_key(x[i]);
          if ((all || k > floor) && (at == 24 || k >> (at + 8) == prefix >> (at + 8))) atomicAdd(&hist[k >> at & 255], value(x[i]));
        }
        __syncthreads();
        if (t == 0) {
          u64 run = sum;
          int b = 255;
          while (b > 0 && run + hist[b] < want) run += hist[b--];
          found = b;
          above = run;
        }
        __syncthreads();
        prefix |= found << at;
        sum = above;
      }
      *over = sum;
      return prefix;
    };
    u64 ties = ~0ull;  // tokens of the last key that stay
    if (r.top_k > 0) {
      u64 over;
      last = select([](float) { return (u64)1; }, (u64)r.top_k, 0u, true, &over);
      ties = (u64)r.top_k - over;
    }
    if (r.top_p < 1.0f) {
      u64 wt = 0, same = 0;
      for (int i = t; i < n; i += NT) {
        const unsigned k = sort_key(x[i]);
        if (k > last) wt += weigh(x[i]);
        same += k == last;
      }
      const u64 over = block_sum(wt, part);
      same = min(block_sum(same, part), ties);
      const u64 one = last ? weigh(key_value(last)) : 0;
      const u64 want = max((u64)1, (u64)__double2ll_ru((double)r.top_p * (double)(over + same * one)));
      if (over < want) {
        ties = min(same, one ? (want - over + one - 1) / one : same);
      } else {
        u64 before;
        last = select([&](float v) { return weigh(v); }, want, last, false, &before);
        const u64 each_one = max((u64)1, weigh(key_value(last)));
        ties = (want - before + each_one - 1) / each_one;
      }
    }
    // the index of the last of the ties
    const int per = (n + NT - 1) / NT, from = min(n, t * per), to = min(n, from + per);
    u64 same = 0, all;
    for (int i = from; i < to; ++i) same += sort_key(x[i]) == last;
    const u64 rank = block_before(same, part, &all);
    if (t == 0) found = UINT_MAX;
    __syncthreads();
    if (rank < ties && rank + same >= ties) {
      u64 left = ties - rank;
      for (int i = from; i < to; ++i)
        if (sort_key(x[i]) == last && --left == 0) found = (unsigned)i;
    }
    __syncthreads();
    last_at = found;
    // and the slices' sums, which the list would have had
    for (int i = 0; i < w.slices; ++i) {
      u64 sum = 0;
      for (int j = i * w.length + t; j < min(n, (i + 1) * w.length); j += NT) {
        const unsigned k = sort_key(x[j]);
        if (k > last || (k == last && (unsigned)j <= last_at)) sum += weigh.least(x[j]);
      }
      sum = block_sum(sum, part);
      if (t == 0) s.kept[i] = sum;
    }
    __syncthreads();
    __threadfence_block();
  } else if (listed > 0) {
    // sorted: falling keys, rising indexes
    int size = (int)listed;
    if (size <= 2 * NT) {
      // by each one's rank: none is there twice
      u64 mine[2];
      int rank[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) mine[j] = t + j * NT < size ? s.list[t + j * NT] : 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) list[t + j * NT] = mine[j];
      __syncthreads();
      const ulonglong2 *const two = reinterpret_cast<const ulonglong2 *>(list);
      for (int i = 0; i < (size + 1) / 2; ++i) {
        const ulonglong2 v = two[i];
#pragma unroll
        for (int j = 0; j < 2; ++j) rank[j] += (v.x > mine[j]) + (v.y > mine[j]);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (t + j * NT < size) list[rank[j]] = mine[j];
    } else {
      while (size & (size - 1)) size += size & -size;
      for (int i = t; i < size; i += NT) list[i] = i < (int)listed ? s.list[i] : 0;
      for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
          __syncthreads();
          for (int i = t; i < size / 2; i += NT) {
            const int at = 2 * i - (i & (j - 1)), to = at + j;
            const u64 p = list[at], q = list[to];
            if ((p < q) == ((at & k) == 0)) {
              list[at] = q;
              list[to] = p;
            }
          }
        }
    }
    __syncthreads();
    // (a thread's run of the sorted list)
    const int per = (size + NT - 1) / NT, from = min((int)listed, t * per), to = min((int)listed, from + per);
    auto value_at = [&](int i) { return key_value((unsigned)(list[i] >> 32)); };
    int end = (int)listed;  // tokens of the list that top-k keeps
    if (r.k < BINS) {
      // (those of bin k are the list's last)
      u64 in = 0, all;
      for (int i = from; i < to; ++i) in += bin_of(value_at(i), r.top, r.per_bin) == r.k;
      block_before(in, part, &all);
      end = (int)listed - (int)all + r.need_k;
    }
    int stop = end;
    if (r.top_p < 1.0f) {
      // the sum that top-p is of: the bins before k, and what is kept of k (or all)
      u64 in = 0, all, sum = 0;
      for (int i = from; i < min(to, end); ++i) {
        const u64 p = weigh(value_at(i));
        sum += p;
        if (r.k < BINS && bin_of(value_at(i), r.top, r.per_bin) == r.k) in += p;
      }
      block_before(in, part, &all);
      const u64 whole = r.k < BINS ? r.before_k + all : r.whole;
      const u64 want = max((u64)1, (u64)__double2ll_ru((double)r.top_p * (double)whole));
      // (bins between hi and k are not in the list, nor does top-p end there)
      u64 total;
      const u64 up = block_before(sum, part, &total);
      if (t == 0) found = (unsigned)end;
      __syncthreads();
      u64 run = r.before_lo + up;
      for (int i = from; i < min(to, end); ++i) {
        const u64 p = weigh(value_at(i));
        if (run < want && run + p >= want) found = (unsigned)i + 1;
        run += p;
      }
      __syncthreads();
      stop = (int)found;
    }
    const u64 final = list[stop - 1];
    last = (unsigned)(final >> 32);
    last_at = ~(unsigned)final;
    __syncthreads();
  }
  // The slices' sums with the list's kept tokens, and the draw.
  u64 *const sums = hist;  // (up to 256 slices)
  for (int i = t; i < w.slices; i += NT) sums[i] = s.kept[i];
  __syncthreads();
  if (listed <= LIST)
    for (int i = t; i < (int)listed; i += NT) {
      const unsigned k = (unsigned)(list[i] >> 32), at = ~(unsigned)list[i];
      if (k > last || (k == last && at <= last_at)) {
        const u64 p = weigh.least(key_value(k));
        if (p) atomicAdd(&sums[at / w.length], p);
      }
    }
  __syncthreads();
  u64 total;
  const u64 mine = t < w.slices ? sums[t] : 0, up = block_before(mine, part, &total);
  // (u times the sum rounds to what may be the sum itself: then the last of them)
  const u64 draw = min((u64)((double)r.u * (double)total), total - 1);
  if (t < w.slices && draw >= up && draw < up + mine) {
    ends[0] = (u64)t;
    ends[1] = up;
  }
  __syncthreads();
  const int begin = (int)ends[0] * w.length, finish = min(n, begin + w.length);
  const int per = (w.length + NT - 1) / NT, from = min(finish, begin + t * per), to = min(finish, from + per);
  auto kept = [&](int i) {
    const float v = x[i];
    const unsigned k = sort_key(v);
    return k > last || (k == last && (unsigned)i <= last_at) ? weigh.least(v) : (u64)0;
  };
  u64 sum = 0, unused;
  for (int i = from; i < to; ++i) sum += kept(i);
  u64 run = ends[1] + block_before(sum, part, &unused);
  if (draw < run || draw >= run + sum) return;
  for (int i = from; i < to; ++i) {
    const u64 p = kept(i);
    run += p;
    if (run > draw) {
      answer(i, (float)((double)p / (double)total));
      return;
    }
  }
}

// Slices of at least 4096 logits, for about two workgroups a CU.
static void sample_slices(int rows, int vocab, int *slices, int *length) {
  int n = std::max(1, std::min({(vocab + 4095) / 4096, (512 + rows - 1) / rows, 128}));
  *length = ((vocab + n - 1) / n + 1023) & ~1023;
  *slices = (vocab + *length - 1) / *length;
}

// Rows of one round of launches: their workspaces take some hundred megabytes at most.
constexpr int kRowsAtOnce = 2048;

size_t sample_workspace(int rows, int vocab) {
  int slices, length;
  sample_slices(std::min(rows, kRowsAtOnce), vocab, &slices, &length);
  return (size_t)std::min(rows, kRowsAtOnce) * row_bytes(slices);
}

hipError_t launch_sample(hipStream_t st, const SampleArgs &all, void *workspace) {
  int bits = 0;
  while (((long)1 << bits) < all.vocab) ++bits;
  SampleWork w;
  w.space = (char *)workspace;
  // (sums stay below 2^62, weights below 2^52)
  w.shift = std::min(62 - bits, 51);
  sample_slices(std::min(all.rows, kRowsAtOnce), all.vocab, &w.slices, &w.length);
  for (int first = 0; first < all.rows; first += kRowsAtOnce) {
    SampleArgs a = all;
    a.rows = std::min(kRowsAtOnce, all.rows - first);
    a.x += (long)first * a.vocab;
    a.u += first;
    if (a.d_temperature) a.d_temperature += first;
    if (a.d_top_k) a.d_top_k += first;
    if (a.d_top_p) a.d_top_p += first;
    if (a.d_min_p) a.d_min_p += first;
    a.tokens += first;
    if (a.probs) a.probs += first;
    const dim3 grid(w.slices, a.rows);
    hipLaunchKernelGGL(sample_ends_kernel, grid, dim3(NT), 0, st, a, w);
    hipLaunchKernelGGL(sample_bins_kernel, grid, dim3(NT), 0, st, a, w);
    hipLaunchKernelGGL(sample_cut_kernel, dim3(a.rows), dim3(NT), 0, st, a, w);
    hipLaunchKernelGGL(sample_list_kernel, grid, dim3(NT), 0, st, a, w);
    hipLaunchKernelGGL(sample_draw_kernel, dim3(a.rows), dim3(NT), 0, st, a, w);
  }
  return hipGetLastError();
}

}  // namespace spissa
