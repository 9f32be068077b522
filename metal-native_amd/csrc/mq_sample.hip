// Drawing a token from a row of logits.
//
// With M the row's largest logit the weights are w(x) = exp((x - M) / T).  The
// tokens in order (largest logit first, ties by index) are cut to a first part of
// them: top_k; of those, with S their weights' sum, the ones before which less
// than top_p S has gone; the ones of w >= min_p.  So what stays is the tokens
// over a logit, and of those that have just it the ones up to an index.  Drawn is
// the first of them, by index, with which their running sum passes u times their
// sum.
//
// A token is a whole number: between two that border on each other in the running
// sum nothing is half right, and 150 thousand borders lie in a row.  Weights are
// therefore taken in 64 bits and summed as whole multiples of 2^-shift (2^-44 for
// 152064 tokens): sums of whole numbers do not depend on their order, which
// atomics and any split of the work change.
//
// The logit at which a cut falls is found digit by digit (11, 11 and 10 bits of
// the logits' order as whole numbers): how many tokens and how much weight each
// value of a digit has, among those that share the digits before it.
#include "mq_device.hpp"
#include "mq_sample.hpp"

#include "../../include/metal_native_amd.h"

namespace mq {
namespace {

constexpr int kThreads = 1024;

template <typename E> __device__ __forceinline__ float to_float(E v) { return (float)v; }

// Whole numbers in the order of the values: NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kNone = 0x007fffffu;   // order_of(-inf)

struct Settings {
  double inv_t, top_p, min_p;
  int64_t top_k;
  bool greedy;
  float u;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& p, int row) {
  Settings s;
  const float t = p.temperatures ? p.temperatures[row] : p.temperature;
  const int k = p.top_ks ? p.top_ks[row] : p.top_k;
  s.top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  const float least = p.min_ps ? p.min_ps[row] : p.min_p;
  s.min_p = least > 0.f ? fminf(least, 1.f) : 0.f;
  s.greedy = !(t > 0.f);
  s.inv_t = 1.0 / (double)t;
  s.top_k = k > 0 && k < p.vocab ? k : p.vocab;
  const float u = p.u[row];
  s.u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  return s;
}

// of the whole workgroup, on every thread
template <typename V, typename F> __device__ __forceinline__ V reduce(V v, V* lds, F&& f) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o; o >>= 1) v = f(v, (V)__shfl_xor(v, o));
  __syncthreads();
  if (lane == 0) lds[w] = v;
  __syncthreads();
  v = lds[0];
  for (int i = 1; i < kThreads / 64; ++i) v = f(v, lds[i]);
  return v;
}
// inclusive, and the sum of all
template <typename V> __device__ __forceinline__ V scan(V v, V* lds, V& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V t = __shfl_up(v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 63) lds[w] = v;
  __syncthreads();
  V before = 0;
  all = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < w) before += lds[i];
    all += lds[i];
  }
  return v + before;
}

typedef unsigned long long ull;

template <typename E> __global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs p, int shift) {
  __shared__ uint32_t cnt[2048];
  __shared__ ull wt[2048], red[kThreads / 64];
  __shared__ struct {
    uint32_t bin;
    ull above_n, above_w;
  } found;
  const int tid = threadIdx.x, row = blockIdx.x, V = p.vocab;
  const E* x = (const E*)p.logits + (int64_t)row * p.ld;
  const Settings st = settings_of(p, row);
  auto key = [&](int i) { return order_of(to_float(x[i])); };

  uint32_t top = 0;
  for (int i = tid; i < V; i += kThreads) top = max(top, key(i));
  top = (uint32_t)reduce<ull>(top, red, [](ull a, ull b) { return a > b ? a : b; });
  if (top <= kNone) {
    if (tid == 0) {
      p.token[row] = -1;
      if (p.logprob) p.logprob[row] = -INFINITY;
    }
    return;
  }
  if (st.greedy) {
    ull first = ~0ull;
    for (int i = tid; i < V && first == ~0ull; i += kThreads)
      if (key(i) == top) first = i;
    first = reduce<ull>(first, red, [](ull a, ull b) { return a < b ? a : b; });
    if (tid == 0) {
      p.token[row] = (int64_t)first;
      if (p.logprob) p.logprob[row] = 0.f;
    }
    return;
  }
  const double M = value_of(top);
  auto real = [&](uint32_t k) { return k == top ? 1.0 : exp(((double)value_of(k) - M) * st.inv_t); };
  auto whole = [&](uint32_t k) { return (ull)__double2ull_rn(ldexp(real(k), shift)); };

  // The key in whose group the n-th token (by_count) or the weight n lies, as
  // counted from the largest; how many tokens and how much weight come before the
  // group, and how many tokens it has.  All of it if there is less.
  struct Cut {
    uint32_t key;
    ull before_n, before_w, n;
  };
  auto find = [&](bool by_count, ull n) {
    Cut c{0, 0, 0, 0};
    int have = 0;
    for (int level = 0; level < 3; ++level) {
      const int bits = level == 2 ? 10 : 11, low = 32 - have - bits;
      for (int i = tid; i < 2048; i += kThreads) cnt[i] = 0, wt[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t k = key(i);
        if (k > kNone && (have == 0 || k >> (32 - have) == c.key)) {
          const uint32_t d = (k >> low) & ((1u << bits) - 1);
          atomicAdd(&cnt[d], 1u);
          atomicAdd(&wt[d], whole(k));
        }
      }
      __syncthreads();
      // digits from the largest down, two to a thread
      const int d0 = 2047 - 2 * tid, d1 = d0 - 1;
      const ull c0 = cnt[d0], c1 = cnt[d1], w0 = wt[d0], w1 = wt[d1];
      ull all;
      const ull cs = scan<ull>(c0 + c1, red, all) - c0 - c1 + c.before_n, end_n = all + c.before_n;
      const ull ws = scan<ull>(w0 + w1, red, all) - w0 - w1 + c.before_w, end_w = all + c.before_w;
      const ull aim = by_count ? min(n, end_n) : min(n, end_w);   // some group reaches it
      auto mine = [&](ull bn, ull bw, ull dn, ull dw) {
        const ull b = by_count ? bn : bw, d = by_count ? dn : dw;
        return b < aim && b + d >= aim;
      };
      if (mine(cs, ws, c0, w0)) found = {(uint32_t)d0, cs, ws};
      if (mine(cs + c0, ws + w0, c1, w1)) found = {(uint32_t)d1, cs + c0, ws + w0};
      __syncthreads();
      c.key = c.key << bits | found.bin;
      c.before_n = found.above_n;
      c.before_w = found.above_w;
      c.n = cnt[found.bin];
      have += bits;
      __syncthreads();
    }
    return c;
  };

  // tokens over the key stay, and the first `ties` of those that have it
  uint32_t at = kNone;
  ull ties = 0, ties_of = 0, kept_w = 0;
  bool cut = false;
  auto take = [&](const Cut& c, ull n) {
    at = c.key;
    ties = n;
    ties_of = c.n;
    cut = true;
  };
  if (st.top_k < V) {
    const Cut c = find(true, st.top_k);
    const ull n = min((ull)st.top_k - c.before_n, c.n);
    take(c, n);
    kept_w = c.before_w + n * whole(c.key);
  }
  if (st.top_p < 1.0) {
    if (!cut) {
      ull sum = 0;
      for (int i = tid; i < V; i += kThreads)
        if (const uint32_t k = key(i); k > kNone) sum += whole(k);
      scan<ull>(sum, red, kept_w);
    }
    const ull aim = max((ull)1, (ull)ceil(fmax(st.top_p, 0.0) * (double)kept_w));
    const Cut c = find(false, aim);
    const ull w = whole(c.key), n = w ? (aim - c.before_w - 1) / w + 1 : c.n;
    // never more than top_k left: a group that it cuts has its ties already
    const bool same = cut && c.key == at;
    take(c, min(n, same ? ties : c.n));
  }
  // the last index among the ties that stay
  int last = V;
  if (cut && ties < ties_of) {
    ull seen = 0;
    for (int i0 = 0; i0 < V; i0 += kThreads) {
      const int i = i0 + tid;
      const bool tie = i < V && key(i) == at;
      ull all;
      const ull r = scan<ull>(tie, red, all) + seen;
      if (tie && r == ties) found.bin = i;
      seen += all;
      if (seen >= ties) break;
    }
    __syncthreads();
    last = (int)found.bin;
  }
  auto weight = [&](int i) -> ull {
    const uint32_t k = key(i);
    if (k <= kNone || (cut && (k < at || (k == at && i > last)))) return 0;
    return real(k) < st.min_p ? 0 : whole(k);
  };
  ull sum = 0, total;
  for (int i = tid; i < V; i += kThreads) sum += weight(i);
  scan<ull>(sum, red, total);
  const ull aim = (ull)floor((double)st.u * (double)total);
  ull before = 0;
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const ull w = i < V ? weight(i) : 0;
    ull all;
    const ull r = scan<ull>(w, red, all) + before;
    if (w && r > aim && r - w <= aim) {
      const uint32_t k0 = key(i);
      p.token[row] = i;
      if (p.logprob) p.logprob[row] = (float)((k0 == top ? 0.0 : ((double)value_of(k0) - M) * st.inv_t) - log(ldexp((double)total, -shift)));
    }
    before += all;
    if (before > aim) break;
  }
}

}  // namespace

size_t sample_workspace(const SampleArgs&, int) { return 0; }

hipError_t sample_launch(const SampleArgs& a, int, void*, hipStream_t s) {
  int shift = 62;
  while ((int64_t)1 << (62 - shift) < a.vocab) --shift;
  if (a.dtype == MQ_SAMPLE_F32) sample_kernel<float><<<a.rows, kThreads, 0, s>>>(a, shift);
  else if (a.dtype == MQ_SAMPLE_BF16) sample_kernel<__bf16><<<a.rows, kThreads, 0, s>>>(a, shift);
  else sample_kernel<_Float16><<<a.rows, kThreads, 0, s>>>(a, shift);
  return hipGetLastError();
}

}  // namespace mq
