// sampler.hip -- one token of each row of logits: temperature, top-k, top-p and
// min-p, and a given random number.
//
// All three filters keep the first tokens in the order of falling logits (equal ones
// by index), so what is kept is known by its last token. Weights w = exp((x - max) / T)
// are formed in 64 bits and held as the nearest whole numbers of 2^-shift: no sum adds an
// error, whatever its order, and a limit lies off the definition's by the weights' own half
// steps alone, n * 2^-(shift + 1) of the largest weight at most (n tokens: 2^-29 for 128256,
// 2^-27 for 2^18, 2^-19 for 2^22, if all round the same way). (Sums in single precision
// would move the borders of some hundred thousand tokens by 2^-24, and one row in a hundred
// would come out another token.)
//
// A row's logits are read three times, by workgroups of a slice each (sample_ends_kernel,
// sample_bins_kernel, sample_list_kernel):
//   1. the slice's largest and smallest logit;
//   2. the counts (for top-k) or else the weights (for top-p) of 1024 bins of (max - x),
//      fine enough that few tokens share the bin in which the filter ends;
//   3. with that bin known: into a list the tokens that have to be put in order (all of
//      the top-k's bins, or those of the bin where top-p ends), and the sums of the
//      weights certain to be kept, by granules of 256 logits.
// Then a workgroup a row (sample_draw_kernel) finds the last kept token in the list (of
// some hundred), draws, and walks the granule in which the draw falls. A row whose list
// would not fit (thousands of tokens in a thousandth of the logits' range, or a top-k of
// thousands) is done in the same way over the whole row. Without filters the third launch
// is left out, and up to 12288 logits are one workgroup's from start to end
// (sample_row_kernel).
//
// Bound by latency for a few rows (one of 128256 logits, all filters: 18 us, four launches
// of 4 to 6 us each); for many by reads and by the weights' 35 operations in 64 bits a
// token: 64 rows of 128256 with settings of their own 43 to 52 us (9, 15, 14, 15 us a launch;
// 33 MB), five rows of 262144 without filters 15 us.
#include <algorithm>
#include <climits>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

typedef unsigned long long u64;

constexpr int NT = 512, BINS = 1024, LIST = 8192, GRANULE = 256, FEW = 256;

// Bits that rise with the value; both zeros alike.
__device__ __forceinline__ unsigned sort_key(float x) {
  const unsigned b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

// A token as a number that falls along the order: its logit's key, then its index.
__device__ __forceinline__ u64 token_of(float x, int i) { return (u64)sort_key(x) << 32 | ~(unsigned)i; }
__device__ __forceinline__ float logit_of(u64 token) { return key_value((unsigned)(token >> 32)); }
__device__ __forceinline__ int index_of(u64 token) { return (int)~(unsigned)token; }

// exp((x - max) / T) as 2^y, y = n + r, |r| <= 1/2, by twelve terms of exp(r ln 2): off by
// at most (1 + |y|) * 2^-51 of itself, as y and log2(e) / T are rounded (half of that the most
// of 6000 formed on the host).
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
  // The nearest whole number of 2^-shift (below 2^52: the sum's low bits are it), or 0 below `least`.
  __device__ __forceinline__ u64 operator()(float x, double least) const {
    const double w = real(x, shift);
    return w >= least ? (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull : 0;
  }
};

// A slice's largest logit with its first place, its smallest, and whether one is NaN or +infinite.
struct Slice {
  float most, least;
  int at, bad;
};
// (by value: the compiler puts what a choice takes by reference into scratch memory)
__device__ __forceinline__ Slice joined(Slice a, Slice b) {
  const int at = b.most > a.most ? +b.at : b.most == a.most ? min(a.at, b.at) : +a.at;
  return Slice{fmaxf(a.most, b.most), fminf(a.least, b.least), at, a.bad | b.bad};
}
// What a row's later passes go by.
struct Row {
  u64 whole, before;  // weights of all, and of the bins before lo; for top-k counts, and those before hi
  float top, per_bin;
  float temperature, top_p, min_p, u;
  int top_k;          // 0: all
  int state;          // kBad..
  int lo, hi;         // bins of the list; tokens of those before lo are certain of all but min_p
  int first;          // the largest logit's first place
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

// The sum of the lanes' values up to this one's, and of all.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_of(u64 v) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_up_to(u64 v) {
  v += dpp_of<0x111, 0xf>(v);  // within a row of 16 lanes, from 1, 2, 4 and 8 before
  v += dpp_of<0x112, 0xf>(v);
  v += dpp_of<0x114, 0xf>(v);
  v += dpp_of<0x118, 0xf>(v);
  v += dpp_of<0x142, 0xa>(v);  // a row's last to the next row
  v += dpp_of<0x143, 0xc>(v);  // the first half's last to the second half
  return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ u64 wave_sum(u64 v) { return last_lane(wave_up_to(v)); }

// The granules of a slice by waves: f(index, logit) for a lane's four, 64 apart, then
// done(granule).
template <class F, class G>
__device__ __forceinline__ void each(const float *x, int from, int to, F f, G done) {
  constexpr int STEP = NT / 64 * GRANULE;
  const int lane = threadIdx.x & 63;
  float next[4];
  auto load = [&](int g) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) next[j] = x[min(g + 64 * j + lane, to - 1)];
  };
  int g = from + (int)(threadIdx.x >> 6) * GRANULE;
  if (g < to) load(g);
  for (; g < to; g += STEP) {
    float v[4] = {next[0], next[1], next[2], next[3]};
    if (g + STEP < to) load(g + STEP);
    if (g + GRANULE <= to) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f(g + 64 * j + lane, v[j]);
    } else {
#pragma unroll 1
      for (int i = g + lane; i < to; i += 64) {
        f(i, v[0]);
        v[0] = v[1];
        v[1] = v[2];
        v[2] = v[3];
      }
    }
    done(g / GRANULE);
  }
}

__device__ __forceinline__ u64 wave_least(u64 v) {
  v = ~v;  // (lane shifts bring zeros where there is no lane)
  v = max(v, dpp_of<0x111, 0xf>(v));
  v = max(v, dpp_of<0x112, 0xf>(v));
  v = max(v, dpp_of<0x114, 0xf>(v));
  v = max(v, dpp_of<0x118, 0xf>(v));
  v = max(v, dpp_of<0x142, 0xa>(v));
  v = max(v, dpp_of<0x143, 0xc>(v));
  return ~last_lane(v);
}

__device__ __forceinline__ u64 block_sum(u64 v, u64 *part) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 r = 0;
  for (int i = 0; i < NT / 64; ++i) r += part[i];
  return r;
}

// The sum of the threads' values before this one's, and of all.
__device__ __forceinline__ u64 block_before(u64 v, u64 *part, u64 *all) {
  const u64 run = wave_up_to(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = run;
  __syncthreads();
  u64 before = 0, total = 0;
  for (int i = 0; i < NT / 64; ++i) {
    if (i < (int)(threadIdx.x >> 6)) before += part[i];
    total += part[i];
  }
  *all = total;
  return before + run - v;
}

// A row's share of the workspace.
struct Space {
  Row *row, *cut;   // before and after the filters' bin is known
  unsigned *listed; // tokens of the list (beyond LIST: not all of them there)
  u64 *list;        // [LIST]: key, and the index's complement
  u64 *bins;        // [BINS] weights or, half as long, counts
  u64 *kept;        // [granules]: weights certain to be kept
  Slice *slices;
};
struct SampleWork {
  char *space;
  size_t row_bytes;
  int slices, length;  // of a row; logits of a slice
  int granules;
  int shift;
};
constexpr size_t kRowHead = 80;  // of each of the two
static_assert(sizeof(Row) <= kRowHead && kRowHead % 16 == 0, "a row's head");
inline size_t row_bytes(int slices, int granules) {
  return 2 * kRowHead + 16 + LIST * 8 + BINS * 8 + (size_t)slices * sizeof(Slice) + ((size_t)granules * 8 + 15) / 16 * 16;
}
__device__ __forceinline__ Space space_of(const SampleWork &w, int row) {
  char *const p = w.space + row * w.row_bytes;
  Space s;
  s.row = reinterpret_cast<Row *>(p);
  s.cut = reinterpret_cast<Row *>(p + kRowHead);
  s.listed = reinterpret_cast<unsigned *>(p + 2 * kRowHead);
  s.list = reinterpret_cast<u64 *>(p + 2 * kRowHead + 16);
  s.bins = s.list + LIST;
  s.slices = reinterpret_cast<Slice *>(s.bins + BINS);
  s.kept = reinterpret_cast<u64 *>(s.slices + w.slices);
  return s;
}

// The ends of x[from, to), for every thread; keep(index, logit) sees each once.
template <class K>
__device__ __forceinline__ Slice ends_of(const float *x, int from, int to, K keep) {
  __shared__ Slice part[NT / 64];
  Slice s{NEG_INF, __builtin_inff(), INT_MAX, 0};
  auto see = [&](int i, float v) __attribute__((always_inline)) {
    s.bad |= !(v < __builtin_inff());
    if (v > s.most) {
      s.most = v;
      s.at = i;
    }
    s.least = fminf(s.least, v);
    keep(i, v);
  };
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
#pragma unroll 2
    for (int i = from + 4 * (int)threadIdx.x; i + 4 <= to; i += 4 * NT) {
      const float4 v = *reinterpret_cast<const float4 *>(x + i);
      see(i, v.x);
      see(i + 1, v.y);
      see(i + 2, v.z);
      see(i + 3, v.w);
    }
    // (a lane's place of the last three; slices begin at multiples of four)
    const int i = (to & ~3) + (int)threadIdx.x;
    if (i < to) see(i, x[i]);
  } else {
#pragma unroll 4
    for (int i = from + (int)threadIdx.x; i < to; i += NT) see(i, x[i]);
  }
  for (int d = 32; d > 0; d >>= 1)
    s = joined(s, Slice{__shfl_xor(s.most, d), __shfl_xor(s.least, d), __shfl_xor(s.at, d), __shfl_xor(s.bad, d)});
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  for (int i = 0; i < NT / 64; ++i) s = joined(s, part[i]);
  return s;
}

// What is to be done for a row of these ends.
__device__ __forceinline__ Row row_of(const SampleArgs &a, const Slice &e, int row) {
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
  r.first = e.at;
  r.whole = r.before = 0;
  r.lo = r.hi = 0;
  return r;
}

// The bins of the list, for r.lo and what follows from it: by the thread that holds, of
// two bins each, the one where the filter ends.
__device__ __forceinline__ void cut(const Row &r, const u64 (&in)[2], u64 *part, Row &to) {
  u64 whole;
  u64 up = block_before(in[0] + in[1], part, &whole);
  // (the last bin of a range cut at 40 temperatures holds no weight: with fewer tokens
  // before it than top-k keeps, those are all that count)
  const bool far = r.per_bin * (40.0f * r.temperature) <= BINS;
  const u64 want = r.top_k > 0 ? (u64)r.top_k : max((u64)1, (u64)__double2ll_ru((double)r.top_p * (double)whole));
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int b = 2 * (int)threadIdx.x + j;
    if (up < want && up + in[j] >= want) {
      to.lo = r.top_k > 0 ? 0 : b;
      to.hi = r.top_k > 0 && b == BINS - 1 && far ? BINS - 2 : b;
      to.before = up;
      to.whole = whole;
    }
    up += in[j];
  }
}

}  // namespace

// The slices' ends; clears the bins. Reads at 4 TB/s (64 rows of 128256: 33 MB in 9 us).
// Grid: (slices, rows).
__global__ __launch_bounds__(NT) void sample_ends_kernel(const SampleArgs a, const SampleWork w) {
  const int row = blockIdx.y, from = blockIdx.x * w.length, to = min(a.vocab, from + w.length);
  const Slice s = ends_of(a.x + (long)row * a.vocab, from, to, [](int, float) {});
  const Space space = space_of(w, row);
  if (threadIdx.x == 0) space.slices[blockIdx.x] = s;
  for (int i = blockIdx.x * NT + threadIdx.x; i < BINS; i += w.slices * NT) space.bins[i] = 0;
}

// The counts or weights of the slice's bins; without a filter the sums of its granules'
// kept weights. Slices' bins meet in memory (one array a slice and a launch a row that
// summed them: 2.6 us more for one row, 1.4 for 64). Grid: (slices, rows).
__global__ __launch_bounds__(NT) void sample_bins_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ u64 weights[BINS];
  const int row = blockIdx.y, from = blockIdx.x * w.length, to = min(a.vocab, from + w.length);
  const float *const x = a.x + (long)row * a.vocab;
  const Space s = space_of(w, row);
  Slice e{NEG_INF, __builtin_inff(), INT_MAX, 0};
  if ((int)(threadIdx.x & 63) < w.slices) e = s.slices[threadIdx.x & 63];
  for (int d = 16; d > 0; d >>= 1)
    e = joined(e, Slice{__shfl_xor(e.most, d), __shfl_xor(e.least, d), __shfl_xor(e.at, d), __shfl_xor(e.bad, d)});
  // (the first half of the wave has them all)
  e = Slice{__shfl(e.most, 0), __shfl(e.least, 0), __shfl(e.at, 0), __shfl(e.bad, 0)};
  const Row r = row_of(a, e, row);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *s.listed = 0;
    *s.row = r;
    *s.cut = r;
  }
  if (r.state < kAll) return;
  const Weigh weigh = weigh_of(r, w.shift);
  const bool by_count = r.top_k > 0, sums = r.state == kAll;
  unsigned *const counts = reinterpret_cast<unsigned *>(weights);
  for (int i = threadIdx.x; i < BINS; i += NT) weights[i] = 0;
  __syncthreads();
  if (by_count) {
    each(x, from, to, [&](int, float v) { atomicAdd(&counts[bin_of(v, r.top, r.per_bin)], 1u); }, [](int) {});
  } else {
    u64 sum = 0;
    each(
        x, from, to,
        [&](int, float v) {
          const u64 p = weigh(v, sums ? weigh.min_p : 0.0);
          sum += p;
          // (what has no weight, far down, would only meet in the last bin)
          if (!sums && p) atomicAdd(&weights[bin_of(v, r.top, r.per_bin)], p);
        },
        [&](int g) {
          if (!sums) return;
          sum = wave_sum(sum);
          if ((threadIdx.x & 63) == 0) s.kept[g] = sum;
          sum = 0;
        });
    if (sums) return;
  }
  __syncthreads();
  // (whole numbers: the order of the slices changes nothing)
  for (int i = threadIdx.x; i < BINS; i += NT) {
    if (by_count) {
      if (counts[i]) atomicAdd(reinterpret_cast<unsigned *>(s.bins) + i, counts[i]);
    } else {
      if (weights[i]) atomicAdd(&s.bins[i], weights[i]);
    }
  }
}

// The bin where the filter ends (by every workgroup for itself), the list's tokens, and the
// sums of the granules' certain ones. Grid: (slices, rows).
__global__ __launch_bounds__(NT) void sample_list_kernel(const SampleArgs a, const SampleWork w) {
  constexpr unsigned HERE = 2048;
  __shared__ u64 list[HERE], part[NT / 64];
  __shared__ unsigned listed, place;
  __shared__ Row ends;
  static_assert(BINS == 2 * NT, "a thread has two bins");
  const int row = blockIdx.y, from = blockIdx.x * w.length, to = min(a.vocab, from + w.length);
  const float *const x = a.x + (long)row * a.vocab;
  const Space s = space_of(w, row);
  // (counts lie in the first half of the bins)
  const ulonglong2 weights = reinterpret_cast<const ulonglong2 *>(s.bins)[threadIdx.x];
  const uint2 counts = reinterpret_cast<const uint2 *>(s.bins)[threadIdx.x];
  Row r = *s.row;
  if (r.state != kList) return;
  const u64 in[2] = {r.top_k > 0 ? (u64)counts.x : weights.x, r.top_k > 0 ? (u64)counts.y : weights.y};
  cut(r, in, part, ends);
  __syncthreads();
  r.lo = ends.lo;
  r.hi = ends.hi;
  r.before = ends.before;
  r.whole = ends.whole;
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.cut = r;
  const Weigh weigh = weigh_of(r, w.shift);
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  u64 sum = 0;
  each(
      x, from, to,
      [&](int i, float v) {
        const int b = bin_of(v, r.top, r.per_bin);
        if (b < r.lo) {
          sum += weigh(v, weigh.min_p);
        } else if (b <= r.hi) {
          const u64 token = token_of(v, i);
          unsigned at = atomicAdd(&listed, 1u);
          if (at < HERE) {
            list[at] = token;
          } else if ((at = atomicAdd(s.listed, 1u)) < LIST) {
            s.list[at] = token;
          }
        }
      },
      [&](int g) {
        if (__any(sum != 0)) sum = wave_sum(sum);
        if ((threadIdx.x & 63) == 0) s.kept[g] = sum;
        sum = 0;
      });
  __syncthreads();
  const unsigned here = min(listed, HERE);
  if (threadIdx.x == 0) place = here ? atomicAdd(s.listed, here) : 0;
  __syncthreads();
  for (unsigned i = threadIdx.x; i < here; i += NT)
    if (place + i < LIST) s.list[place + i] = list[i];
}

struct Select {
  u64 sums[256], both[NT / 64][2], found, above;
  unsigned counts[256], alone;
};
// The first token, from the largest down, at which the running sum of value(token), from
// `base` on, reaches `want`. all(f): f(token) for the thread's tokens. Eight bits a
// round, from the first in which any two differ, until one token is left.
template <class All, class Value>
__device__ __forceinline__ u64 select(All all, Value value, u64 want, u64 base, Select &s) {
  const int t = threadIdx.x;
  u64 any = 0, every = ~0ull;
  all([&](u64 e) {
    any |= e;
    every &= e;
  });
  for (int d = 32; d > 0; d >>= 1) {
    any |= __shfl_xor(any, d);
    every &= __shfl_xor(every, d);
  }
  __syncthreads();
  if ((t & 63) == 0) {
    s.both[t >> 6][0] = any;
    s.both[t >> 6][1] = every;
  }
  __syncthreads();
  for (int i = 0; i < NT / 64; ++i) {
    any |= s.both[i][0];
    every &= s.both[i][1];
  }
  int top = 64 - __clzll((long long)(any ^ every));  // undecided bits
  if (any == every) return any;
  u64 prefix = top == 64 ? 0 : any >> top;
  while (top > 0) {
    const int shift = max(0, top - 8);
    const unsigned digits = (1u << (top - shift)) - 1;
    if (t < 256) {
      s.sums[t] = 0;
      s.counts[t] = 0;
    }
    __syncthreads();
    all([&](u64 e) {
      if ((top == 64 ? 0 : e >> top) != prefix) return;
      const unsigned d = (unsigned)(e >> shift) & digits;
      const u64 v = value(e);
      if (v) atomicAdd(&s.sums[d], v);
      atomicAdd(&s.counts[d], 1u);
    });
    __syncthreads();
    if (t < 64) {  // a lane's four digits, the largest in lane 0
      u64 v[4], four = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) four += v[i] = s.sums[255 - 4 * t - i];
      u64 run = base + wave_up_to(four) - four;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (run < want && run + v[i] >= want) {
          s.found = 255 - 4 * t - i;
          s.above = run;
          s.alone = s.counts[255 - 4 * t - i];
        }
        run += v[i];
      }
    }
    __syncthreads();
    prefix = prefix << (top - shift) | s.found;
    base = s.above;
    top = shift;
    if (s.alone == 1) {
      __syncthreads();
      all([&](u64 e) {
        if (e >> top == prefix) s.found = e;
      });
      __syncthreads();
      return s.found;
    }
  }
  return prefix;
}

// (a function of its own: a kernel that runs once waits for each line of its code)
__device__ __attribute__((noinline)) u64 weigh_apart(Weigh weigh, float x, double least) { return weigh(x, least); }
// A token's share of the kept weights, its own as it was before it became a whole number (of
// a token 27 temperatures down that is one or two of 2^-40 with 2^22 logits).
__device__ __attribute__((noinline)) float share_of(Weigh weigh, float x, u64 total) {
  return (float)(weigh.real(x, weigh.shift) / (double)total);
}

// What a workgroup needs to find the last kept token.
struct alignas(16) Choice {
  u64 part[NT / 64], bins[BINS], few[FEW + 32], values[FEW + 32], runs[FEW], ends[2];
  unsigned ranks[FEW], many;
  int bin;
  Select select;
};
// The last kept token of a row from its list (in LDS, not yet waited for), or, where it is
// not whole, from all of its logits, at(index).
template <class W, class A>
__device__ __forceinline__ u64 last_kept(const Row &r, W weigh, const u64 *list, int listed, bool fits, int n, A at,
                                         Choice &c) {
  const int t = threadIdx.x;
  // The tokens of few[] before each of them, and their values' sum: a thread's share of
  // the pairs, and what they come to for token t.
  unsigned rank;
  u64 run;
  auto order = [&](int m) {
    const int share = (m + 4 * NT / 64 - 1) / (4 * NT / 64) * 4, from = (t >> 6) * share;  // of a wave
    if (t >= m && t < NT / 64 * share) c.few[t] = 0;  // (before none)
    __syncthreads();
    for (int j = t & 63; j < m; j += 64) {
      const u64 e = c.few[j];
      unsigned before = 0;
      u64 sum = 0;
#pragma unroll 2
      for (int i = from; i < from + share; i += 4) {
        const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(c.few + i), b = *reinterpret_cast<const ulonglong2 *>(c.few + i + 2);
        const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(c.values + i), y = *reinterpret_cast<const ulonglong2 *>(c.values + i + 2);
        before += (a.x > e) + (a.y > e) + (b.x > e) + (b.y > e);
        sum += (a.x > e ? x.x : 0) + (a.y > e ? x.y : 0) + (b.x > e ? y.x : 0) + (b.y > e ? y.y : 0);
      }
      atomicAdd(&c.ranks[j], before);
      atomicAdd(&c.runs[j], sum);
    }
    __syncthreads();
    rank = t < m ? c.ranks[t] : 0;
    run = t < m ? c.runs[t] : 0;
  };
  auto least_of = [&](u64 v) {
    v = wave_least(v);
    __syncthreads();
    if ((t & 63) == 0) c.part[t >> 6] = v;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) v = min(v, c.part[i]);
    return v;
  };
  auto clear = [&]() {
    if (t < FEW) {
      c.ranks[t] = 0;
      c.runs[t] = 0;
    }
    if (t == 0) c.many = 0;
  };
  auto part_of = [&](u64 whole) { return max((u64)1, (u64)__double2ll_ru((double)r.top_p * (double)whole)); };
  clear();
  __syncthreads();
  if (listed <= FEW) {  // both filters at once
    u64 p = 0, token = 0;
    if (t < listed) {
      c.few[t] = token = list[t];
      c.values[t] = p = weigh(logit_of(token), 0.0);
    }
    __syncthreads();
    order(listed);
    const bool in = t < listed && (r.top_k == 0 || rank < (unsigned)r.top_k);
    const u64 whole = r.top_k > 0 ? block_sum(in ? p : 0, c.part) : r.whole;
    const bool kept = in && (r.top_p >= 1.0f || (r.top_k > 0 ? 0 : r.before) + run < part_of(whole));
    return least_of(kept ? token : ~0ull);
  }
  // Top-k's last token, then top-p's of what that leaves: each in a bin that is known or
  // found, and of that bin's (of all, where the list is not whole) among few, or by bits of
  // the order. (With fewer listed than top-k keeps, no other token has weight: see cut().)
  u64 last = 0;
  int bin = fits ? r.hi : -1;
  auto left = [&](auto f) __attribute__((always_inline)) {
    const int count = fits ? listed : n;
#pragma unroll 1
    for (int i = t; i < count; i += NT) {
      const u64 e = fits ? list[i] : token_of(at(i), i);
      if (e >= last && (bin < 0 || bin_of(logit_of(e), r.top, r.per_bin) == bin)) f(e);
    }
  };
#pragma unroll 1
  for (int filter = 0; filter < 2; ++filter) {
    if (filter == 0 ? r.top_k == 0 || (fits && listed < r.top_k) : r.top_p >= 1.0f) continue;
    u64 want = (u64)r.top_k, base = fits ? r.before : 0;
    if (filter == 1) {
      u64 whole = r.whole;
      if (!fits || r.top_k > 0) {
        bin = -1;
        for (int i = t; i < BINS; i += NT) c.bins[i] = 0;
        __syncthreads();
        left([&](u64 e) {
          const u64 p = weigh(logit_of(e), 0.0);
          if (p) atomicAdd(&c.bins[bin_of(logit_of(e), r.top, r.per_bin)], p);
        });
        __syncthreads();
        const u64 in[2] = {c.bins[2 * t], c.bins[2 * t + 1]};
        u64 up = block_before(in[0] + in[1], c.part, &whole);
        want = part_of(whole);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (up < want && up + in[j] >= want) {
            c.bin = 2 * t + j;
            c.ends[0] = up;
          }
          up += in[j];
        }
        __syncthreads();
        bin = c.bin;
        base = c.ends[0];
      }
      want = part_of(whole);
    }
    left([&](u64 e) {
      const unsigned place = atomicAdd(&c.many, 1u);
      if (place < FEW) {
        c.few[place] = e;
        c.values[place] = filter == 0 ? 1 : weigh(logit_of(e), 0.0);
      }
    });
    __syncthreads();
    const unsigned m = c.many;
    if (m <= FEW) {
      order((int)m);
      last = least_of(t < (int)m && base + run < want ? c.few[t] : ~0ull);
    } else {
      last = select(left, [&](u64 e) { return filter == 0 ? 1 : weigh(logit_of(e), 0.0); }, want, base, c.select);
    }
    __syncthreads();
    clear();
    __syncthreads();
  }
  return last;
}

// Whether a row is answered already (and, if so, its answer).
__device__ __forceinline__ bool answered(const SampleArgs &a, const Row &r, int row) {
  if (r.state != kBad && r.state != kGreedy) return false;
  if (threadIdx.x == 0) {
    if (r.state == kBad) atomicOr(a.err, kDevErrSampling);
    a.tokens[row] = r.state == kBad ? -1 : r.first;
    if (a.probs) a.probs[row] = r.state == kBad ? 0.0f : 1.0f;
  }
  return true;
}
// (u times the sum rounds to what may be the sum itself: then the last of them)
__device__ __forceinline__ u64 drawn(const Row &r, u64 total) {
  return min((u64)((double)r.u * (double)total), total - 1);
}

// The last kept token, the draw, and the token. A chain of loads and sums over the
// workgroup: 5.6 us with up to 256 listed, 15 with a thousand in an end bin of equal ones.
// Grid: rows.
__global__ __launch_bounds__(NT) void sample_draw_kernel(const SampleArgs a, const SampleWork w) {
  __shared__ u64 list[LIST], sums[NT];
  __shared__ Choice choice;
  const int row = blockIdx.x, t = threadIdx.x, n = a.vocab;
  const float *const x = a.x + (long)row * n;
  const Space s = space_of(w, row);
  // (loads that wait for none: the row, the list's first tokens, a thread's run of granules)
  const Row r = *s.cut;
  const unsigned written = *s.listed;
  const u64 token = s.list[t];
  const int per = (w.granules + NT - 1) / NT, g0 = min(w.granules, t * per), g1 = min(w.granules, g0 + per);
  u64 mine = 0;
  for (int g = g0; g < g1; ++g) mine += s.kept[g];
  if (answered(a, r, row)) return;
  const Weigh weigher = weigh_of(r, w.shift);
  auto weigh = [&](float v, double least) { return weigh_apart(weigher, v, least); };
  const double min_p = weigher.min_p;
  const int listed = r.state == kList ? (int)min(written, LIST + 1u) : 0;
  const bool fits = listed <= LIST;
  u64 last = 0;  // of the kept tokens
  if (r.state == kList) {
    list[t] = token;
    if (fits)
      for (int i = t + NT; i < listed; i += NT) list[i] = s.list[i];
    last = last_kept(r, weigh, list, listed, fits, n, [&](int i) { return x[i]; }, choice);
    if (!fits) {  // the granules' sums, which the list would have completed
      u64 sum = 0;
      each(
          x, 0, n,
          [&](int i, float v) {
            if (token_of(v, i) >= last) sum += weigh(v, min_p);
          },
          [&](int g) {
            sum = wave_sum(sum);
            if ((t & 63) == 0) s.kept[g] = sum;
            sum = 0;
          });
      __threadfence_block();
      __syncthreads();
      mine = 0;
      for (int g = g0; g < g1; ++g) mine += s.kept[g];
    }
  }
  // Threads' runs of granules, with the list's kept tokens, and the draw.
  sums[t] = mine;
  __syncthreads();
  auto each_listed = [&](auto see) {  // (in the list and kept)
    for (int i = t; fits && i < listed; i += NT)
      if (list[i] >= last) {
        const u64 p = weigh(logit_of(list[i]), min_p);
        if (p) see(index_of(list[i]) / GRANULE, p);
      }
  };
  each_listed([&](int g, u64 p) { atomicAdd(&sums[g / per], p); });
  __syncthreads();
  u64 total;
  mine = sums[t];
  const u64 up = block_before(mine, choice.part, &total);
  const u64 draw = drawn(r, total);
  if (draw >= up && draw < up + mine) {
    choice.ends[0] = (u64)t;
    choice.ends[1] = up;
  }
  __syncthreads();
  // The granule of that thread's.
  const int first = (int)choice.ends[0] * per;
  u64 run = choice.ends[1];
  if (per > 1) {
    for (int i = t; i < per; i += NT) sums[i] = first + i < w.granules ? s.kept[first + i] : 0;
    __syncthreads();
    each_listed([&](int g, u64 p) {
      if (g >= first && g < first + per) atomicAdd(&sums[g - first], p);
    });
    __syncthreads();
  }
  if (t >= 64) return;
  int g = 0;
  while (g + 1 < per && run + sums[g] <= draw) run += sums[g++];
  // Its logits, 64 at a time.
  const int from = (first + g) * GRANULE + t;
  float v[GRANULE / 64];
#pragma unroll
  for (int j = 0; j < GRANULE / 64; ++j) v[j] = x[min(from + 64 * j, n - 1)];
#pragma unroll 1
  for (int i = from, j = 0; j < GRANULE / 64; ++j, i += 64) {
    const u64 p = i < n && token_of(v[0], i) >= last ? weigh(v[0], min_p) : 0;
    const u64 sum = run + wave_up_to(p);
    if (sum > draw && sum - p <= draw) {
      a.tokens[row] = i;
      if (a.probs) a.probs[row] = share_of(weigher, v[0], total);
    }
    run = last_lane(sum);
    if (run > draw) return;
#pragma unroll
    for (int k = 1; k < GRANULE / 64; ++k) v[k - 1] = v[k];
  }
}

// All of it for rows of at most ROW logits, held in LDS, a workgroup each: the same steps
// over the same numbers, four neighbours a thread at a time. Bound by latency and by one
// CU's operations in 64 bits (kRow has the times). Grid: rows.
template <int ROW>
__global__ __launch_bounds__(NT) void sample_row_kernel(const SampleArgs a, const int shift) {
  constexpr int HERE = 1536;  // (with 12288 logits 79 KB: two workgroups a CU)
  constexpr int WAVE = 256;   // logits of a wave's turn
  static_assert(ROW <= 64 * WAVE, "a granule a lane");
  __shared__ __attribute__((aligned(16))) float held[ROW];
  __shared__ u64 list[HERE], sums[64];
  __shared__ Choice c;
  __shared__ Row found;
  __shared__ unsigned written;
  const int row = blockIdx.x, t = threadIdx.x, n = a.vocab;
  for (int i = t; i < BINS; i += NT) c.bins[i] = 0;
  if (t < 64) sums[t] = 0;
  if (t == 0) written = 0;
  const Slice e = ends_of(a.x + (long)row * n, 0, n, [&](int i, float v) { held[i] = v; });
  Row r = row_of(a, e, row);
  if (answered(a, r, row)) return;
  const Weigh weigher = weigh_of(r, shift);
  auto weigh = [&](float v, double least) { return weigh_apart(weigher, v, least); };
  // f(index, its four logits), of which those from n on do not count
  auto fours = [&](int from, auto f) __attribute__((always_inline)) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(held + from);
    f(from, v);
  };
  u64 last = 0;
  if (r.state == kList) {
    unsigned *const counts = reinterpret_cast<unsigned *>(c.bins);
#pragma unroll 1
    for (int from = 4 * t; from < n; from += 4 * NT)
      fours(from, [&](int i, f32x4 v) __attribute__((always_inline)) {
        if (r.top_k > 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (i + j < n) atomicAdd(&counts[bin_of(v[j], r.top, r.per_bin)], 1u);
        } else {
          u64 p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = weigher(v[j], 0.0);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (i + j < n && p[j]) atomicAdd(&c.bins[bin_of(v[j], r.top, r.per_bin)], p[j]);
        }
      });
    __syncthreads();
    u64 in[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) in[j] = r.top_k > 0 ? counts[2 * t + j] : c.bins[2 * t + j];
    cut(r, in, c.part, found);
    __syncthreads();
    r.lo = found.lo;
    r.hi = found.hi;
    r.before = found.before;
    r.whole = found.whole;
#pragma unroll 1
    for (int from = 4 * t; from < n; from += 4 * NT)
      fours(from, [&](int i, f32x4 v) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int b = bin_of(v[j], r.top, r.per_bin);
          if (i + j < n && b >= r.lo && b <= r.hi) {
            const unsigned at = atomicAdd(&written, 1u);
            if (at < HERE) list[at] = token_of(v[j], i + j);
          }
        }
      });
    __syncthreads();
    const int listed = (int)written;
    last = last_kept(r, weigh, list, listed, listed <= HERE, n, [&](int i) { return held[i]; }, c);
  }
  // The waves' sums of kept weights, the draw and its wave's turn.
  auto kept = [&](int i, f32x4 v, u64 (&p)[4]) __attribute__((always_inline)) {
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = i + j < n && token_of(v[j], i + j) >= last ? weigher(v[j], weigher.min_p) : 0;
      sum += p[j];
    }
    return sum;
  };
  u64 p[4];
#pragma unroll 1
  for (int from = 4 * t; from - 4 * (t & 63) < n; from += 4 * NT)
    fours(from, [&](int i, f32x4 v) __attribute__((always_inline)) {
      const u64 sum = kept(i, v, p);
      if (!__any(sum != 0)) return;
      const u64 all = wave_sum(sum);
      if ((t & 63) == 0) sums[i / WAVE] = all;
    });
  __syncthreads();
  if (t >= 64) return;
  const u64 mine = sums[t], up = wave_up_to(mine), total = last_lane(up), draw = drawn(r, total);
  const int g = __ffsll((unsigned long long)__ballot(draw < up)) - 1;
  const u64 before = __shfl(up - mine, g);
  fours(WAVE * g + 4 * t, [&](int i, f32x4 v) __attribute__((always_inline)) {
    u64 run = kept(i, v, p);
    run = before + wave_up_to(run) - run;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (run <= draw && run + p[j] > draw) {
        a.tokens[row] = i + j;
        if (a.probs) a.probs[row] = share_of(weigher, v[j], total);
      }
      run += p[j];
    }
  });
}

// Longest row that one workgroup takes. (One row of 1000, 4096, 8192 and 12288 logits with
// all filters: 8, 10, 12 and 14 us against 15, 17, 18 and 17 in slices; by top-p alone 8, 11,
// 15 and 19 us against 16, 19, 20 and 19; 1024 rows of 12288: 39 us against 56.)
constexpr int kRow = 12288;

// Rows of one round of launches: their workspaces take some hundred megabytes at most.
constexpr int kRowsAtOnce = 1024;

// Slices of 4096 logits or more, up to 32 a row, for up to four workgroups a CU (64 rows of
// 128256: 49.6 us, with two 53.2, with eight the same; one row, five rows of 262144: 20.0 and
// 16.2 us, with up to 16 slices 21.4 and 19.9).
static SampleWork sample_work(int rows, int vocab) {
  SampleWork w{};
  rows = std::min(rows, kRowsAtOnce);
  const int n = std::max(1, std::min({(vocab + 4095) / 4096, (1024 + rows - 1) / rows, 32}));
  w.length = ((vocab + n - 1) / n + 1023) & ~1023;
  w.slices = (vocab + w.length - 1) / w.length;
  w.granules = (vocab + GRANULE - 1) / GRANULE;
  w.row_bytes = row_bytes(w.slices, w.granules);
  int bits = 0;
  while (((long)1 << bits) < vocab) ++bits;
  w.shift = std::min(62 - bits, 51);  // (sums stay below 2^62, weights below 2^52)
  return w;
}

size_t sample_workspace(int rows, int vocab) {
  if (vocab <= kRow) return 0;
  return (size_t)std::min(rows, kRowsAtOnce) * sample_work(rows, vocab).row_bytes;
}

hipError_t launch_sample(hipStream_t st, const SampleArgs &all, void *workspace) {
  SampleWork w = sample_work(all.rows, all.vocab);
  w.space = (char *)workspace;
  const bool filters = all.d_top_k || all.d_top_p || all.top_p < 1.0f || (all.top_k > 0 && all.top_k < all.vocab);
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
    if (a.vocab <= kRow) {
      hipLaunchKernelGGL((sample_row_kernel<kRow>), dim3(a.rows), dim3(NT), 0, st, a, w.shift);
      continue;
    }
    const dim3 grid(w.slices, a.rows);
    hipLaunchKernelGGL(sample_ends_kernel, grid, dim3(NT), 0, st, a, w);
    hipLaunchKernelGGL(sample_bins_kernel, grid, dim3(NT), 0, st, a, w);
    if (filters) hipLaunchKernelGGL(sample_list_kernel, grid, dim3(NT), 0, st, a, w);
    hipLaunchKernelGGL(sample_draw_kernel, dim3(a.rows), dim3(NT), 0, st, a, w);
  }
  return hipGetLastError();
}

}  // namespace spissa
