// sampler.hip -- one token of each row of logits: temperature, top-k, top-p and
// min-p, and a given random number.
//
// All three filters keep the first tokens in the order of falling logits (equal ones
// by index), so what is kept is known by a logit and how many tokens of just that
// logit stay. Weights w = exp((x - max) / T) are formed in 64 bits and held as whole
// numbers of 2^-shift: their sums are exact, whatever the order, and the limits are
// met where the definition has them (sums in single precision would move the borders
// of some hundred thousand tokens by 2^-24, and one row in a hundred would come out
// another token).
#include <climits>

#include "internal.hpp"
#include "lanes.hpp"

namespace spissa {

namespace {

typedef unsigned long long u64;

// Bits that rise with the value; both zeros alike.
__device__ __forceinline__ unsigned sort_key(float x) {
  const unsigned b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

struct Weigh {
  double top, inv, unit, min_p;  // unit: 2^shift
  __device__ __forceinline__ double real(float x) const { return exp(((double)x - top) * inv); }
  __device__ __forceinline__ u64 fixed(double w) const { return (u64)__double2ll_rn(w * unit); }
  __device__ __forceinline__ u64 operator()(float x) const { return fixed(real(x)); }
  __device__ __forceinline__ u64 least(float x) const {  // 0 below min_p
    const double w = real(x);
    return w >= min_p ? fixed(w) : 0;
  }
};

constexpr int NT = 1024;

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

}  // namespace

// A workgroup a row.
__global__ __launch_bounds__(NT) void sample_kernel(const SampleArgs a, int shift) {
  __shared__ u64 hist[256], part[NT / 64];
  __shared__ unsigned found;
  __shared__ u64 above;
  const int row = blockIdx.x, t = threadIdx.x, n = a.vocab;
  const float *const x = a.x + (long)row * n;
  const float temperature = a.d_temperature ? a.d_temperature[row] : a.temperature;
  const float top_p = a.d_top_p ? a.d_top_p[row] : a.top_p, min_p = a.d_min_p ? a.d_min_p[row] : a.min_p;
  const int top_k = a.d_top_k ? a.d_top_k[row] : a.top_k;
  const float u = a.u[row];

  float big = NEG_INF;
  bool bad = false;
  for (int i = t; i < n; i += NT) {
    bad |= !(x[i] < __builtin_inff());
    big = fmaxf(big, x[i]);
  }
  for (int d = 32; d > 0; d >>= 1) big = fmaxf(big, __shfl_xor(big, d));
  __shared__ float bigs[NT / 64];
  if ((t & 63) == 0) bigs[t >> 6] = big;
  bad = __syncthreads_or(bad);
  for (int i = 0; i < NT / 64; ++i) big = fmaxf(big, bigs[i]);
  bad |= big == NEG_INF || !(u >= 0.0f && u < 1.0f) || !(temperature >= 0.0f && temperature < __builtin_inff()) ||
         !(top_p >= 0.0f && top_p <= 1.0f) || !(min_p >= 0.0f && min_p <= 1.0f);
  if (bad) {
    if (t == 0) {
      atomicOr(a.err, kDevErrSampling);
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = 0.0f;
    }
    return;
  }
  const bool greedy = temperature == 0.0f;
  const Weigh weigh{(double)big, greedy ? 1.0 : 1.0 / (double)temperature, ldexp(1.0, shift), (double)min_p};

  // The last kept logit's key, and how many tokens of it stay.
  unsigned last = 0;
  int ties = INT_MAX;
  // Eight bits a round, the highest first: the key at which the running sum from
  // above (of `value` over keys above `floor`) reaches `want`, and what is above it.
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
  if (greedy) {
    last = sort_key(big);
    ties = 1;
  } else {
    if (top_k > 0 && top_k < n) {
      u64 over;
      last = select([](float) { return (u64)1; }, (u64)top_k, 0u, true, &over);
      ties = top_k - (int)over;
    }
    if (top_p < 1.0f) {
      u64 w = 0, total;
      int same = 0;
      for (int i = t; i < n; i += NT) {
        const unsigned k = sort_key(x[i]);
        if (k > last) w += weigh(x[i]);
        same += k == last;
      }
      const u64 over = block_sum(w, part);
      same = min((int)block_sum((u64)same, part), ties);
      const u64 one = weigh(key_value(last));
      total = over + (u64)same * one;
      const u64 want = max((u64)1, (u64)__double2ll_ru((double)top_p * (double)total));
      if (over < want) {
        ties = min(same, (int)min((u64)INT_MAX, one ? (want - over + one - 1) / one : (u64)INT_MAX));
      } else {
        u64 before;
        last = select([&](float v) { return weigh(v); }, want, last, false, &before);
        const u64 each = max((u64)1, weigh(key_value(last)));
        ties = (int)min((u64)INT_MAX, (want - before + each - 1) / each);
      }
    }
  }

  // In index order: a thread's range, its place among the ties, its kept weights.
  const int per = (n + NT - 1) / NT, from = min(n, t * per), to = min(n, from + per);
  u64 same = 0, all;
  for (int i = from; i < to; ++i) same += sort_key(x[i]) == last;
  const u64 rank = block_before(same, part, &all);
  auto walk = [&](auto see) {
    u64 r = rank;
    for (int i = from; i < to; ++i) {
      const unsigned k = sort_key(x[i]);
      if (k < last || (k == last && r++ >= (u64)ties)) continue;
      if (see(i, greedy ? weigh.fixed(1.0) : weigh.least(x[i]))) return;
    }
  };
  u64 kept = 0, total;
  walk([&](int, u64 w) {
    kept += w;
    return false;
  });
  const u64 before = block_before(kept, part, &total);
  // (u times the sum rounds to what may be the sum itself: then the last of them)
  const u64 at = min((u64)((double)u * (double)total), total - 1);
  if (at < before || at >= before + kept) return;
  u64 run = before;
  walk([&](int i, u64 w) {
    run += w;
    if (run <= at) return false;
    a.tokens[row] = i;
    if (a.probs) a.probs[row] = (float)((double)w / (double)total);
    return true;
  });
}

hipError_t launch_sample(hipStream_t st, const SampleArgs &a) {
  int bits = 0;
  while (((long)1 << bits) < a.vocab) ++bits;
  // (sums stay below 2^62, weights within a double's whole numbers)
  const int shift = 62 - bits < 51 ? 62 - bits : 51;
  hipLaunchKernelGGL(sample_kernel, dim3(a.rows), dim3(NT), 0, st, a, shift);
  return hipGetLastError();
}

}  // namespace spissa
