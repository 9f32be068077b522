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
// therefore taken in 64 bits (to 4e-14 of themselves), and what is drawn goes by
// their sums as whole multiples of a unit: 2^-44, in rows of more than 2^18 tokens
// coarser (2^-40 at 2^22), of a short top_k's list 2^-50.  Whole numbers add up to the
// same in any order, and halves of a row that hold the same logits to the same half.
// Tokens of less than half a unit are never drawn.  The sums by which top_p cuts are
// floating ones of 64 bits (units where top_p alone cuts, and on the long way), grouped
// by parts: how a row is dealt out can move a cut that lies within their rounding, and
// nothing else.
//
// A row is dealt out to `parts` workgroups, a wave taking 1024 tokens at a time
// (a sub).  What a row needs follows from its settings, which the GPU alone may
// know (Kind); the launches are the same for all of them:
//   scan    of every part: its largest logit, and by kind its first token; the
//           largest logit of each lane of a sub; or how many tokens lie in each cell
//           of a grid over the logits.
//   bounds  where the grid was filled: from all parts' grids, the logits between
//           which the cuts must fall.
//   gather  the subs' sums of what lies over these (where nothing but min_p cuts, of
//           all), and a list of the tokens between them.
//   pick    the cuts among the listed tokens (or those of the lanes that may hold
//           the first top_k), the sub in which the running sum passes its aim, and the
//           token in it.
// The grid only says where to look: that a cut falls among the listed tokens is
// checked with the weights' sums.  Where it does not, or a list is too short, the row
// goes the long way: cuts found digit by digit by one workgroup, pass after pass.  Such
// rows are those with masses of equal logits at a cut (more of a part's than kListRow /
// parts, or for a short top_k of more than kFewRoom lanes: a mask of the type's lowest
// value that leaves fewer tokens than top_k, where one of -inf does not), those whose
// cut by top_p lies under 2^-28 of the largest weight, and those of infinite logits.
//
// Bound by the issue of instructions: a row is read twice, and 63 million weights of 20
// instructions in 64 bits take longer than their bytes.  152064 logits, us of a call: one
// row, top_k 50 and top_p 0.9, 14.6 (latency of some ten barriers and as many reads behind
// one another); 416 rows of fp16, top_p 0.95, 156 (scan 45, bounds 14, gather 80, pick 21;
// read once they would take 25); 64 of bf16, settings of each, 69; 48 x 32003 in fp32,
// min_p 0.05, 17.  The plain form (a sort, sums, searches) takes 410, 8700, 2000 and 620.
// The long way, 1, 64 and 416 rows of fp16: 20 tokens over a mask of the lowest value,
// top_k 50, 820, 827 and 1644 (masked by -inf 15, 18 and 42); all logits equal, top_p 0.5,
// 988, 1107 and 2259; one token with nearly all of the weight, top_p 0.9999, 231, 265 and 555.
#include "mq_device.hpp"
#include "mq_sample.hpp"

#include "../../include/metal_native_amd.h"

#include <cfloat>

#include <algorithm>

namespace mq {
namespace {

typedef unsigned long long ull;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kSub = 1024;
constexpr int kListRow = 4096;   // list entries of a row, over all parts
constexpr int kAtOnce = 4;       // weights that a lane takes at the same time: registers for eight waves on a SIMD
constexpr int kFewMost = 512;    // top_k up to which a row may be kFew

// Whole numbers in the order of the values: NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kNone = 0x007fffffu;   // order_of(-inf)

// How many low bits of order_of follow from the others
template <typename E> constexpr int kLow = 0;
template <> constexpr int kLow<_Float16> = 13;
template <> constexpr int kLow<__bf16> = 16;

enum Kind { kGreedy, kFew, kGrid, kFloor };   // kFloor: nothing, or min_p alone, cuts

struct Settings {
  double inv_t, top_p, min_p;
  int top_k;   // vocab: none
  float u;
  int kind;
};
// few: the largest top_k that goes by the lanes' largest logits
__device__ __forceinline__ Settings settings_of(const SampleArgs& p, int row, int few) {
  Settings s;
  const float t = p.temperatures ? p.temperatures[row] : p.temperature;
  const int k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float least = p.min_ps ? p.min_ps[row] : p.min_p, u = p.u[row];
  s.top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  s.min_p = least > 0.f ? fminf(least, 1.f) : 0.f;
  s.inv_t = 1.0 / (double)t;
  s.top_k = k > 0 && k < p.vocab ? k : p.vocab;
  s.u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  s.kind = !(t > 0.f) || s.top_k == 1 ? kGreedy
           : s.top_k <= few           ? kFew
           : s.top_k < p.vocab || s.top_p < 1.0 ? kGrid : kFloor;
  return s;
}

// ---- weights ----
// w = 2^(t / 64), t = (x - M) 64 log2(e) / T: the nearest whole number of t by
// a table and the exponent's bits, the rest by its series to the fourth power,
// (log(2) / 128)^5 / 120 = 4e-14 of w.  Some 20 instructions where the library's exp
// takes twice as many.
struct Weights {
  const double* table;   // 2^(i / 64)
  double c;
  float M;
  // M finite; 2^-1020 for what is less, for -inf and NaN
  __device__ __forceinline__ double finite(float x) const {
    return at(__builtin_fmax(((double)x - (double)M) * c, -65280.0));
  }
  // 0 for NaN and -inf, and for what is under 2^-1020
  __device__ __forceinline__ double operator()(float x) const {
    const double t = (x == M ? 0.0 : (double)x - (double)M) * c;
    return t >= -65280.0 ? at(t) : 0.0;
  }
  __device__ __forceinline__ double at(double t) const {
    constexpr double kWhole = 0x1.8p52, L = 0.69314718055994530942 / 64;
    const double n = t + kWhole, f = t - (n - kWhole);
    const int i = (int)(uint32_t)__double_as_longlong(n);
    double e = __builtin_fma(f, L * L * L * L / 24, L * L * L / 6);
    e = __builtin_fma(f, e, L * L / 2);
    e = __builtin_fma(f, e, L) * f;
    const double w = table[i & 63];
    typedef int i2 __attribute__((ext_vector_type(2)));
    i2 bits = __builtin_bit_cast(i2, __builtin_fma(w, e, w));
    bits[1] += (i & ~63) << 14;   // i / 64 to the exponent
    return __builtin_bit_cast(double, bits);
  }
};
__device__ __forceinline__ double steps_of(double inv_t) { return inv_t * (64 * 1.44269504088896340736); }
__device__ __forceinline__ void fill_table(double* table) {   // before a barrier
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(threadIdx.x / 64.0);
}
// w as a whole number of units, to the nearest; one = 2^52 units: 2^8 for 2^-44
__device__ __forceinline__ ull whole(double w, double one) { return (ull)(__double_as_longlong(w + one) - __double_as_longlong(one)); }
// of a list's tokens, no more than kListRow of them, in 2^-50
__device__ __forceinline__ ull whole_of_list(double w) { return whole(w, 4.0); }
constexpr double kListUnit = 0x1p-50;
// floor(u n): a whole number passes u n where it passes this
__device__ __forceinline__ ull share_of(float u, ull n) {
  const uint32_t b = __float_as_uint(u), down = 150 - (b >> 23);   // u = m 2^-down < 1
  if (b >> 23 == 0 || down > 100) return 0;
  return (ull)((unsigned __int128)((b & 0x7fffff) | 0x800000) * n >> down);
}

// ---- the grid: cells of 1/128 of a factor of two in weight, the same ones for all
// parts of a row; kFine of them under the largest logit's (28 factors of two: a cut by
// top_p alone that lies further down is not found, as where 150 thousand weights of
// 2^-28, 6e-4 of the largest, are more than top_p leaves out), the rest by eights, what
// lies under all of these in the last one ----
constexpr int kFine = 3584, kCoarse = 4608, kCells = kFine + kCoarse;
constexpr float kEnd = 0x1p29f;   // the grid's ends
__device__ __forceinline__ float grid_scale(double inv_t) {
  return (float)fmin(fmax(inv_t * (128 * 1.44269504088896340736), 1e-30), 1e30);
}
__device__ __forceinline__ int grid_of(float x, float scale) {   // grows with x
  return (int)floorf(__builtin_amdgcn_fmed3f(x * scale, -kEnd, kEnd));
}
__device__ __forceinline__ int coarse_of(int g, int top) { return kFine + min(kCoarse - 1, (top >> 3) - (g >> 3)); }
// The logit at a cell's lower edge, moved `way` by more than its roundings
__device__ __forceinline__ float edge_of(int g, float scale, float way) {
  if (fabsf((float)g) >= kEnd) return way * INFINITY;
  const float x = (float)g / scale;
  return x + way * (fabsf(x) * 0x1p-20f + 0x1p-20f / scale);
}

// ---- sums over a wave, then over the workgroup's first N waves (the others have gone, if there are any) ----
template <typename V> __device__ __forceinline__ V from_lane(V v, int b) {   // of lane ^ b, without the LDS unit
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, xor_lane(__builtin_bit_cast(float, v), b));
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 h = __builtin_bit_cast(f2, v);
    return __builtin_bit_cast(V, (f2){xor_lane(h[0], b), xor_lane(h[1], b)});
  }
}
template <typename V, typename F> __device__ __forceinline__ V wave_reduce(V v, F&& f) {   // on every lane
  v = f(v, from_lane(v, 1));
  v = f(v, from_lane(v, 2));
  v = f(v, from_lane(v, 4));
  v = f(v, from_lane(v, 8));
  v = f(v, from_lane(v, 16));
  return f(v, from_lane(v, 32));
}
template <typename V> __device__ __forceinline__ V wave_sum(V v) {
  return wave_reduce(v, [](V a, V b) { return a + b; });
}
// zero where the lane has no source
template <int CTRL, int ROWS, typename V> __device__ __forceinline__ V shifted(V v) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
  } else {
    typedef int i2 __attribute__((ext_vector_type(2)));
    const i2 h = __builtin_bit_cast(i2, v);
    return __builtin_bit_cast(V, (i2){__builtin_amdgcn_update_dpp(0, h[0], CTRL, ROWS, 0xF, false),
                                      __builtin_amdgcn_update_dpp(0, h[1], CTRL, ROWS, 0xF, false)});
  }
}
template <typename V> __device__ __forceinline__ V wave_scan(V v) {   // inclusive
  v += shifted<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
  v += shifted<0x112, 0xF>(v);
  v += shifted<0x114, 0xF>(v);
  v += shifted<0x118, 0xF>(v);
  v += shifted<0x142, 0xA>(v);   // row_bcast 15, 31
  v += shifted<0x143, 0xC>(v);
  return v;
}
// What the waves exchange, by turns in two halves: one barrier a sum, since who is
// past it has read the half that the next one but one writes.
struct Group {
  ull* lds;   // [2 * kWaves]
  int half = 0;
  // every wave's value, of wave i on the lanes of i % N
  template <int N, typename V> __device__ __forceinline__ V of_waves(V v, int from = 0) {
    half ^= kWaves;
    if ((int)(threadIdx.x & 63) == from) *(V*)(lds + half + (threadIdx.x >> 6)) = v;
    __syncthreads();
    return *(const V*)(lds + half + (threadIdx.x & (N - 1)));
  }
  template <int N, typename V, typename F> __device__ __forceinline__ V reduce(V v, F&& f) {   // on every thread
    v = of_waves<N>(wave_reduce(v, f));
#pragma unroll
    for (int o = 1; o < N; o <<= 1) v = f(v, from_lane(v, o));
    return v;
  }
  template <int N, typename V> __device__ __forceinline__ V sum(V v) {
    return reduce<N>(v, [](V a, V b) { return a + b; });
  }
  template <int N, typename V> __device__ __forceinline__ V least(V v) {
    return reduce<N>(v, [](V a, V b) { return a < b ? a : b; });
  }
  template <int N, typename V> __device__ __forceinline__ V most(V v) {
    return reduce<N>(v, [](V a, V b) { return a > b ? a : b; });
  }
  // of numbers that are the same on a wave's lanes
  template <int N> __device__ __forceinline__ uint32_t sum_of_waves(uint32_t n) {
    n = of_waves<N>(n);
#pragma unroll
    for (int o = 1; o < N; o <<= 1) n += from_lane(n, o);
    return n;
  }
  // inclusive, and the sum of all
  template <int N, typename V> __device__ __forceinline__ V scan(V v, V& all) {
    v = wave_scan(v);
    V t = of_waves<N>(v, 63);   // N waves' sums, again and again
    t += shifted<0x111, 0xF>(t);
    t += shifted<0x112, 0xF>(t);
    if constexpr (N > 4) t += shifted<0x114, 0xF>(t);
    if constexpr (N > 8) t += shifted<0x118, 0xF>(t);
    all = at_lane(t, N - 1);
    return v + at_lane(shifted<0x111, 0xF>(t), (int)(threadIdx.x >> 6));   // of the waves before
  }
  template <typename V> static __device__ __forceinline__ V at_lane(V v, int lane) {
    lane = __builtin_amdgcn_readfirstlane(lane);
    if constexpr (sizeof(V) == 4) {
      return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
      typedef int i2 __attribute__((ext_vector_type(2)));
      const i2 h = __builtin_bit_cast(i2, v);
      return __builtin_bit_cast(V, (i2){__builtin_amdgcn_readlane(h[0], lane), __builtin_amdgcn_readlane(h[1], lane)});
    }
  }
};

// ---- a wave's 1024 tokens ----
template <typename E> struct Row {
  const E* x;
  int V;
  bool aligned;   // its first element to 16 bytes
  __device__ __forceinline__ Row(const SampleArgs& p, int row) : x((const E*)p.logits + (int64_t)row * p.ld), V(p.vocab), aligned(((uintptr_t)x & 15) == 0) {}
  static constexpr int kPer = 16 / sizeof(E);
  // the lane's j-th: index within the sub, growing with j
  __device__ __forceinline__ int at(int j) const { return at(j, threadIdx.x & 63); }
  __device__ __forceinline__ int at(int j, int lane) const {
    return aligned ? j / kPer * (64 * kPer) + lane * kPer + j % kPer : j * 64 + lane;
  }
  struct Part {   // 16-bit tokens two to a register, however they came
    uint32_t w[4 * sizeof(E)];
    __device__ __forceinline__ float operator[](int j) const {
      if constexpr (sizeof(E) == 4) {
        return __uint_as_float(w[j]);
      } else {
        typedef E two __attribute__((ext_vector_type(2)));
        return (float)__builtin_bit_cast(two, w[j / 2])[j % 2];
      }
    }
  };
  __device__ __forceinline__ void load(int sub, Part& p) const {   // -inf past the row
    const int base = sub * kSub, lane = threadIdx.x & 63;
    if (aligned && base + kSub <= V) {
#pragma unroll
      for (int i = 0; i < 16 / kPer; ++i) {
        const u4 t = *(const u4*)(x + base + (i * 64 + lane) * kPer);
#pragma unroll
        for (int k = 0; k < 4; ++k) p.w[4 * i + k] = t[k];
      }
    } else {   // by distances from one place, which are constants
      const E* from = x + (base + at(0));
      const int left = V - base - at(0);
      auto one = [&](int d) -> uint32_t {
        if constexpr (sizeof(E) == 4) return __float_as_uint(d < left ? from[d] : -INFINITY);
        else return __builtin_bit_cast(uint16_t, d < left ? from[d] : (E)-INFINITY);
      };
      auto all = [&](auto&& distance) {
#pragma unroll
        for (int i = 0; i < (int)(4 * sizeof(E)); ++i)
          p.w[i] = sizeof(E) == 4 ? one(distance(i)) : one(distance(2 * i)) | one(distance(2 * i + 1)) << 16;
      };
      if (aligned) all([](int j) { return j / kPer * (64 * kPer) + j % kPer; });
      else all([](int j) { return j * 64; });
    }
  }
  // f(sub, its tokens) for the subs s0, s0 + kWaves .. before s1, the next one's loads on their way
  template <typename F> __device__ __forceinline__ void each(int s0, int s1, F&& f) const {
    Part next;
    if (s0 < s1) load(s0, next);
    for (int s = s0; s < s1; s += kWaves) {
      const Part v = next;
      if (s + kWaves < s1) load(s + kWaves, next);
      f(s, v);
    }
  }
};

// ---- what the launches hand on ----
struct Part {
  float top;        // largest logit
  uint32_t first;   // kGreedy: the first token of that logit
  uint32_t far;     // kGrid, where top_k does not cut: tokens under the fine cells, and what is no number
  uint32_t listed;  // tokens that asked for a place in the list; past its length: it is not whole
  uint32_t over_n;  // kGrid, where top_k cuts: tokens from Bounds::k_hi on
  uint32_t cells;   // kGrid: the last cell that holds a token, and one
  double over_k, over_p;   // kGrid: weight from k_hi on (of all tokens where top_k does not cut), from p_hi on
};
struct Bounds {   // by bounds, for gather and pick: the cut of top_k falls among logits of k_lo <= x < k_hi, that of top_p between p_lo and p_hi
  float k_lo, k_hi, p_lo, p_hi;   // -inf where there is none
  int cut_k, cut_p;
  __device__ __forceinline__ float sure() const { return cut_p ? p_hi : k_hi; }   // tokens from here on stay, but for min_p
};
struct Work {
  Part* part;       // [rows, parts]
  Bounds* bounds;   // [rows]
  ull* sub;         // [rows, subs]
  float* most;      // [rows, subs, 64]: of each lane
  uint32_t* list;   // [rows, parts, places]
  uint32_t* cells;  // [rows, parts, kCells]
  int row0, parts, subs, places, few;
  double one;      // 2^52 of the units of sub
  int part_subs;   // of a part; fewer of the last
  __device__ __forceinline__ int first_sub(int part) const { return min(part * part_subs, subs); }
};

template <typename E> __global__ __launch_bounds__(kThreads, 8) void sample_scan_kernel(SampleArgs p, Work ws) {
  __shared__ ull lds[2 * kWaves];
  Group grp{lds};
  __shared__ uint32_t cells[kCells];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = blockIdx.x / ws.parts, part = blockIdx.x - r * ws.parts, row = ws.row0 + r;
  const Settings st = settings_of(p, row, ws.few);
  const Row<E> x(p, row);
  const int s0 = ws.first_sub(part) + w, s1 = ws.first_sub(part + 1);
  const bool count = st.top_k < p.vocab;
  typedef typename Row<E>::Part Tokens;
  float mine = -INFINITY;
  x.each(s0, s1, [&](int s, const Tokens& v) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = fmaxf(m, v[j]);   // the number of the two, where one is NaN
    if (st.kind == kFew) ws.most[((int64_t)r * ws.subs + s) * 64 + lane] = m;
    mine = fmaxf(mine, m);
  });
  if (st.kind == kGrid)
    for (int i = tid; i < (count ? kCells : kFine + 64); i += kThreads) cells[i] = 0;
  const float M = grp.reduce<kWaves>(mine, [](float a, float b) { return fmaxf(a, b); });
  Part& out = ws.part[(int64_t)r * ws.parts + part];
  if (tid == 0) {
    out.top = M;
    out.cells = 0;
  }
  if (M == -INFINITY || st.kind == kFew || st.kind == kFloor) return;
  if (st.kind == kGreedy) {
    uint32_t first = ~0u;
    Tokens v;
    for (int s = s0; s < s1 && first == ~0u; s += kWaves) {
      x.load(s, v);
#pragma unroll
      for (int j = 15; j >= 0; --j) first = v[j] == M ? s * kSub + x.at(j) : first;
    }
    first = (uint32_t)grp.least<kWaves, ull>(first);
    if (tid == 0) out.first = first;
  } else {
    const float scale = grid_scale(st.inv_t);
    const int top = grid_of(M, scale);
    x.each(s0, s1, [&](int, const Tokens& v) {
      if (!count) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          atomicAdd(&cells[min(top - grid_of(v[j], scale), kFine + lane)], 1u);   // past the fine ones: one for each lane
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int g = grid_of(v[j], scale), d = top - g;
          if (v[j] > -INFINITY) atomicAdd(&cells[d < kFine ? d : coarse_of(g, top)], 1u);
        }
      }
    });
    __syncthreads();
    uint32_t* to = ws.cells + ((int64_t)r * ws.parts + part) * kCells;
    uint32_t end = 0;
    for (int i = tid; i < (count ? kCells : kFine); i += kThreads) {
      const uint32_t c = cells[i];
      to[i] = c;
      if (c) end = i + 1;
    }
    end = (uint32_t)grp.most<kWaves, ull>(end);
    const uint32_t far = wave_sum(cells[kFine + lane]);
    if (tid == 0) {
      out.cells = end;
      out.far = far;   // used where top_k does not cut
    }
  }
}

// The row's largest logit, over its parts (at most kPartsMost: one to a lane)
constexpr int kPartsMost = 16;
__device__ __forceinline__ float top_of(const Part* part, int parts) {
  const int i = threadIdx.x & (kPartsMost - 1);
  float M = i < parts ? part[i].top : -INFINITY;
#pragma unroll
  for (int o = kPartsMost / 2; o; o >>= 1) M = fmaxf(M, from_lane(M, o));
  return M;
}

// All parts' grids laid over each other: a part's cell, from its own largest logit
// down, is one of the row's.  Then between which logits the cuts fall; a workgroup
// for each row, two to a CU (as pick: 416 rows 14 us where one takes 24).
__global__ __launch_bounds__(kThreads, 8) void sample_bounds_kernel(SampleArgs p, Work ws) {
  __shared__ uint32_t numbers[kCells];
  __shared__ ull lds[2 * kWaves];
  Group grp{lds};
  __shared__ double at_k[2];
  __shared__ uint32_t far_of;
  __shared__ int cell;
  const int tid = threadIdx.x, r = blockIdx.x, row = ws.row0 + r;
  const Settings st = settings_of(p, row, ws.few);
  if (st.kind != kGrid) return;
  const Part* parts = ws.part + (int64_t)r * ws.parts;
  const float M = top_of(parts, ws.parts);
  if (M == -INFINITY) return;
  const bool count = st.top_k < p.vocab;
  const int cells = count ? kCells : kFine;
  const float scale = grid_scale(st.inv_t);
  const int top = grid_of(M, scale);
  for (int i = tid; i < cells; i += kThreads) numbers[i] = 0;
  if (tid == 0) {
    far_of = 0;
    cell = cells;
  }
  __syncthreads();
  uint32_t far = 0;   // tokens under the row's fine cells
  // as many threads to each part: a power of two
  int lanes = kThreads;
  while (lanes * ws.parts > kThreads) lanes >>= 1;
  const int of = tid / lanes;
  if (of < ws.parts) {
    const Part& q = parts[of];
    const int end = (int)q.cells, mt = grid_of(q.top, scale), down = top - mt;
    const uint32_t* from = ws.cells + ((int64_t)r * ws.parts + of) * kCells;
    if ((tid & (lanes - 1)) == 0 && !count && end) far += q.far;
    constexpr int kStep = 4;   // loads of a thread on their way, four cells each (the last ones past end: zeros)
    for (int d0 = 4 * (tid & (lanes - 1)); d0 < end; d0 += 4 * kStep * lanes) {
      u4 n4[kStep];
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        const int d = d0 + 4 * k * lanes;
        n4[k] = d < end ? *(const u4*)(from + d) : (u4){0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        const int d = d0 + 4 * k * lanes;
        if (d + down + 3 < kFine && d + 3 < kFine) {
#pragma unroll
          for (int c = 0; c < 4; ++c) atomicAdd(&numbers[d + down + c], n4[k][c]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t n = n4[k][c];
            int to = d + c + down;
            if (d >= kFine) to = kFine + min(kCoarse - 1, d + c - kFine + (top >> 3) - (mt >> 3));
            else if (to >= kFine) to = count ? coarse_of(mt - d - c, top) : -1;
            if (to < 0) far += n;
            else if (n) atomicAdd(&numbers[to], n);
          }
        }
      }
    }
  }
  if (far) atomicAdd(&far_of, far);
  __syncthreads();
  constexpr int N = kCells / kThreads;
  const int per = count ? N : (kFine + kThreads - 1) / kThreads, b0 = per * tid;   // the thread's cells
  double wt[N], mine = 0, low = 0;
  uint32_t mine_n = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int b = b0 + k;
    wt[k] = 0;
    if (k >= per) continue;
    const uint32_t n = b < cells ? numbers[b] : 0;
    // the weight at a fine cell's middle, a coarse one's lower edge; the top cell's is 1
    const float down = b < kFine ? (float)b : (float)(top - 8 * ((top >> 3) - (b - kFine))) + 0.5f;
    wt[k] = (double)((float)n * exp2f(down * (-1.f / 128)));
    mine += wt[k];
    low += b < kFine ? 0 : wt[k];
    mine_n += n;
  }
  double all;
  const double before = grp.scan<kWaves, double>(mine, all) - mine;   // to a few steps of the sum
  if (count) {
    uint32_t all_n, at = grp.scan<kWaves, uint32_t>(mine_n, all_n) - mine_n;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t n = numbers[b0 + k];   // kCells are N to a thread
      if (at < (uint32_t)st.top_k && at + n >= (uint32_t)st.top_k) cell = b0 + k;   // one thread
      at += n;
    }
  }
  __syncthreads();
  const int cell_k = cell;
  int cell_p0 = cells, cell_p1 = cells;
  if (st.top_p < 1.0) {
    // What is known: sums of fine cells to e of themselves (half a cell's width, and the rounding of the product
    // with the scale); coarse ones to 7 / 128 of a factor of two; what lies under the fine cells from nothing to
    // 2^-28 a token; of cell_k some part.
    const double e = 2.8e-3 + fabs((double)top) * 0x1p-28, share = fmax(st.top_p, 0.0);
    const double slack = count ? 0.045 * grp.sum<kWaves, double>(low) : far_of * 0x1p-28;
    double upto = all, in_k = 0;
    if (cell_k < cells) {
      double run = before;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        run += wt[k];
        if (b0 + k == cell_k && k < per) at_k[0] = run, at_k[1] = wt[k];
      }
      __syncthreads();
      upto = at_k[0];
      in_k = at_k[1];
    }
    const double lo = (upto - in_k) * (1 - e), hi = upto * (1 + e) + slack;   // of what top_p is a share of
    double run = before;
    ull may = cells, must = cells;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (k >= per) continue;
      run += wt[k];
      const int b = b0 + k;
      const double rest = fmax(upto - run, 0.0);   // weight past the cell, with all of cell_k
      if (b <= cell_k && wt[k] > 0) {
        if (run * (1 + e) + slack >= share * lo && fmax(rest - in_k, 0.0) * (1 - e) <= (1 - share) * hi) may = min(may, (ull)b);
        if (run * (1 - e) >= share * hi || rest * (1 + e) + slack <= (1 - share) * upto * (1 - e)) must = min(must, (ull)b);
      }
    }
    cell_p1 = (int)grp.least<kWaves, ull>(must);
    cell_p0 = (int)grp.least<kWaves, ull>(may);
  }
  if (tid) return;
  auto lower = [&](int c) { return c < kFine ? top - c : 8 * ((top >> 3) - (c - kFine)); };   // smallest g of a cell
  auto upper = [&](int c) { return c < kFine ? top - c : min(8 * ((top >> 3) - (c - kFine)) + 7, top - kFine); };
  Bounds b{-INFINITY, -INFINITY, -INFINITY, -INFINITY, cell_k < cells, st.top_p < 1.0};
  if (b.cut_k) {
    b.k_hi = edge_of(upper(cell_k) + 1, scale, 1.f);
    b.k_lo = cell_k == kCells - 1 ? -INFINITY : edge_of(lower(cell_k), scale, -1.f);
  }
  if (b.cut_p) {
    b.p_hi = edge_of(upper(min(cell_p0, min(cell_p1, cells - 1))) + 1, scale, 1.f);
    b.p_lo = cell_p1 >= cells || cell_p1 == kCells - 1 ? b.k_lo : edge_of(lower(cell_p1), scale, -1.f);
  }
  ws.bounds[r] = b;
}

template <typename E> __global__ __launch_bounds__(kThreads, 8) void sample_gather_kernel(SampleArgs p, Work ws) {
  __shared__ double table[64];
  __shared__ ull lds[2 * kWaves];
  Group grp{lds};
  __shared__ uint32_t places;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = blockIdx.x / ws.parts, part = blockIdx.x - r * ws.parts, row = ws.row0 + r;
  const Settings st = settings_of(p, row, ws.few);
  if (st.kind != kGrid && st.kind != kFloor) return;
  typedef typename Row<E>::Part Tokens;
  Part* parts = ws.part + (int64_t)r * ws.parts;
  const float M = top_of(parts, ws.parts);
  if (fabsf(M) == INFINITY) return;   // nothing to draw; or the long way
  fill_table(table);
  if (tid == 0) places = 0;
  __syncthreads();
  const Weights weight{table, steps_of(st.inv_t), M};
  const Row<E> x(p, row);
  const int s0 = ws.first_sub(part) + w, s1 = ws.first_sub(part + 1);
  ull* sub = ws.sub + (int64_t)r * ws.subs;
  const double one = ws.one;
  // 16 numbers of w + one as they are, less 16 of one: their units
  const ull none = 16 * (ull)__double_as_longlong(one);
  if (st.kind == kFloor) {
    // weights under min_p, as logits, with a margin for the division by T
    const double span = (log(st.min_p) - 1e-9) / st.inv_t;
    const float low = st.min_p > 0 ? (float)((double)M + span - 1e-9 * fabs(span)) : -INFINITY, least = low - fabsf(low) * 0x1p-22f;
    x.each(s0, s1, [&](int s, const Tokens& v) {
      ull sum = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j % kAtOnce == 0) __builtin_amdgcn_sched_barrier(0);
        if (!__any(v[j] >= least)) continue;
        const double wt = weight.finite(v[j]);
        sum += whole(wt >= st.min_p ? wt : 0.0, one);
        asm volatile("" : "+v"(sum));
      }
      sum = wave_sum(sum);
      if (lane == 0) sub[s] = sum;
    });
    return;
  }
  const Bounds b = ws.bounds[r];
  const bool cut_k = b.cut_k, cut_p = b.cut_p;
  const float sure = b.sure();
  uint32_t* list = ws.list + ((int64_t)r * ws.parts + part) * ws.places;
  double over_k = 0, over_p = 0;
  ull kept_all = 0;
  uint32_t over_n = 0;
  auto enlist = [&](int s, uint32_t take) {   // bit j: the lane's j-th token
    while (take) {
      const int j = __builtin_ctz(take);
      take &= take - 1;
      const uint32_t at = atomicAdd(&places, 1u);
      if (at < (uint32_t)ws.places) list[at] = s * kSub + x.at(j);
    }
  };
  if (!cut_k && st.min_p == 0) {   // top_p alone
    const float lo = fmaxf(b.p_lo, -FLT_MAX);
    x.each(s0, s1, [&](int s, const Tokens& v) {
      ull kept = 0;
      uint32_t take = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j % kAtOnce == 0) __builtin_amdgcn_sched_barrier(0);
        const double wt = weight.finite(v[j]);
        const bool stays = v[j] >= sure;
        over_k += wt;
        kept += (ull)__double_as_longlong((stays ? wt : 0.0) + one);
        take |= ((v[j] >= lo) & !stays) << j;
        if (j % kAtOnce == kAtOnce - 1) asm volatile("" : "+v"(over_k), "+v"(kept), "+v"(take));   // added up here, not at the end
      }
      kept -= none;
      kept_all += kept;
      kept = wave_sum(kept);
      if (lane == 0) sub[s] = kept;
      enlist(s, take);
    });
  } else {
    // where top_k cuts, what lies under both windows has no part in anything
    const float least = cut_k ? (cut_p ? fminf(b.k_lo, b.p_lo) : b.k_lo) : -INFINITY;
    x.each(s0, s1, [&](int s, const Tokens& v) {
      ull kept = 0;
      uint32_t take = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j % kAtOnce == 0) __builtin_amdgcn_sched_barrier(0);
        if (!__any(v[j] >= least)) continue;
        const bool in_k = cut_k & (v[j] >= b.k_lo) & (v[j] < b.k_hi), in_p = cut_p & (v[j] >= b.p_lo) & (v[j] < b.p_hi);
        take |= ((in_k | in_p) & (v[j] > -INFINITY)) << j;
        const double wt = weight.finite(v[j]);
        const bool of_k = !cut_k | (v[j] >= b.k_hi);
        over_k += of_k ? wt : 0.0;
        over_n += of_k;
        const double stays = v[j] >= sure ? wt : 0.0;
        over_p += stays;
        kept += whole(stays >= st.min_p ? stays : 0.0, one);
        asm volatile("" : "+v"(over_k), "+v"(over_p), "+v"(kept), "+v"(take), "+v"(over_n));
      }
      kept = wave_sum(kept);
      if (lane == 0) sub[s] = kept;
      enlist(s, take);
    });
  }
  over_p += (double)kept_all * (one * 0x1p-52);
  over_k = grp.sum<kWaves, double>(over_k);
  over_p = grp.sum<kWaves, double>(over_p);
  const ull n = grp.sum<kWaves, ull>(over_n);
  if (tid == 0) {
    Part& out = parts[part];
    out.listed = places;
    out.over_n = (uint32_t)n;
    out.over_k = over_k;
    out.over_p = over_p;
  }
}

struct LongWay {
  uint32_t cnt[2048];
  ull wt[2048];
  struct {
    uint32_t bin;
    ull above_n, above_w;
  } found;
};

// One workgroup for a row, pass after pass: cuts are found digit by digit (11, 11
// and 10 bits of order_of), from how many tokens and how much weight each value of
// a digit has among those that share the digits before it.
__device__ __forceinline__ void tell(const SampleArgs& p, int row, int token, double log_share) {
  p.token[row] = token;
  if (p.logprob) p.logprob[row] = (float)log_share;
}
template <typename E>
__device__ __forceinline__ void long_way(const SampleArgs& p, int row, const Settings& st, const Weights& weigh, double one, LongWay& sh, Group& grp) {
  uint32_t* const cnt = sh.cnt;
  ull* const wt = sh.wt;
  auto& found = sh.found;
  const int tid = threadIdx.x, V = p.vocab;
  const E* x = (const E*)p.logits + (int64_t)row * p.ld;
  auto key = [&](int i) { return order_of((float)x[i]); };
  auto real = [&](uint32_t k) { return weigh(value_of(k)); };
  auto whole = [&](uint32_t k) { return mq::whole(real(k), one); };

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
      const ull cs = grp.scan<kWaves, ull>(c0 + c1, all) - c0 - c1 + c.before_n, end_n = all + c.before_n;
      const ull ws = grp.scan<kWaves, ull>(w0 + w1, all) - w0 - w1 + c.before_w, end_w = all + c.before_w;
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
      grp.scan<kWaves, ull>(sum, kept_w);
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
      const ull r = grp.scan<kWaves, ull>(tie, all) + seen;
      if (tie && r == ties) found.bin = i;
      seen += all;
      if (seen >= ties) break;
    }
    __syncthreads();
    last = (int)found.bin;
  }
  auto weight = [&](int i) -> ull {
    const uint32_t k = key(i);
    if (k <= kNone || (cut && (k < at || (k == at && i > last))) || real(k) < st.min_p) return 0;
    return whole(k);
  };
  ull sum = 0, total;
  for (int i = tid; i < V; i += kThreads) sum += weight(i);
  total = grp.sum<kWaves, ull>(sum);
  const ull aim = share_of(st.u, total);
  ull before = 0;
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const ull w = i < V ? weight(i) : 0;
    ull all;
    const ull r = grp.scan<kWaves, ull>(w, all) + before;
    if (w && r > aim && r - w <= aim) tell(p, row, i, log(real(key(i)) / ((double)total * (one * 0x1p-52))));
    before += all;
    if (before > aim) break;
  }
}

// ---- the last launch: a workgroup for each row, of which eight waves do the work
// (their barriers are shorter) unless the row goes the long way ----
constexpr int kNear = 8, kNearThreads = 64 * kNear;
constexpr uint32_t kRanked = 192;   // tokens that are put in order by their ranks; more by merging
constexpr int kFewRoom = 1024;   // places for the tokens of kFew that are as large as the top_k-th largest of the lanes'

struct List {
  uint32_t key[kListRow], idx[kListRow];   // order_of without its low bits
  ull units[kListRow];                     // weights in kListUnit
};

// How many of n numbers (a zero behind them) are larger than mine
__device__ __forceinline__ uint32_t rank_of(ull mine, const ull* of, int n) {
  typedef ull ull2 __attribute__((ext_vector_type(2)));
  uint32_t rank = 0;
#pragma unroll 4
  for (int i = 0; i < (n + 1) / 2; ++i) {
    const ull2 q = ((const ull2*)of)[i];
    rank += (q[0] > mine) + (q[1] > mine);
  }
  return rank;
}

// The threads' numbers in falling order over the first N of them: runs that fall and rise
// in turn are merged to longer ones, in a wave by lanes, over waves with one barrier a step.
template <int N> __device__ __forceinline__ ull in_order(ull v, ull (*turn)[kThreads]) {
  const int tid = threadIdx.x;
  int half = 0;
#pragma unroll
  for (int run = 2; run <= N; run <<= 1)
#pragma unroll
    for (int by = run >> 1; by; by >>= 1) {
      ull other;
      if (by < 64) {
        other = from_lane(v, by);
      } else {
        turn[half][tid] = v;
        __syncthreads();
        other = turn[half][tid ^ by];
        half ^= 1;
      }
      const bool larger = ((tid & by) == 0) == ((tid & run) == 0);
      v = (v > other) == larger ? v : other;
    }
  __syncthreads();   // `turn` may be used again
  return v;
}

template <typename F> __device__ __forceinline__ uint32_t number_of(int held, Group& grp, F&& of) {
  uint32_t c = 0;
  for (int i = threadIdx.x; i < (held + 63 & ~63); i += kNearThreads) c += __popcll(__ballot(i < held && of(i)));
  return grp.sum_of_waves<kNear>(c);
}
// For how many entries `of` is true to 1, to 2 and to 3, in 16 bits each
template <typename F> __device__ __forceinline__ ull numbers_of(int held, Group& grp, F&& of) {
  ull c = 0;
  for (int i = threadIdx.x; i < (held + 63 & ~63); i += kNearThreads)
    c += (ull)__popcll(__ballot(i < held && of(i, 1u))) | (ull)__popcll(__ballot(i < held && of(i, 2u))) << 16 |
         (ull)__popcll(__ballot(i < held && of(i, 3u))) << 32;
  c = grp.of_waves<kNear>(c);
#pragma unroll
  for (int o = 1; o < kNear; o <<= 1) c += from_lane(c, o);
  return c;
}
// Of the entries that are true to `of`, the n-th largest key, among `bits` of them
// under a common head, and the n-th smallest index: two bits a barrier
template <typename F>
__device__ __forceinline__ uint32_t nth_key(int held, uint32_t n, uint32_t head, int bits, const uint32_t* key, Group& grp, F&& of) {
  uint32_t least = head;
#pragma unroll 1
  for (int bit = (bits - 1) & ~1; bit >= 0; bit -= 2) {
    const ull c = numbers_of(held, grp, [&](int i, uint32_t d) { return key[i] >= (least | d << bit) && of(i); });
    least |= ((uint32_t)(c >> 32) >= n ? 3u : ((uint32_t)(c >> 16 & 0xffff) >= n ? 2u : ((uint32_t)(c & 0xffff) >= n ? 1u : 0u))) << bit;
  }
  return least;
}
template <typename F>
__device__ __forceinline__ uint32_t nth_index(int held, uint32_t n, int vocab, const uint32_t* idx, Group& grp, F&& of) {
  uint32_t most = 0;   // fewer than n lie under it
#pragma unroll 1
  for (int bit = (31 - __clz(vocab)) & ~1; bit >= 0; bit -= 2) {
    const ull c = numbers_of(held, grp, [&](int i, uint32_t d) { return idx[i] < (most | d << bit) && of(i); });
    most |= ((uint32_t)(c >> 32) < n ? 3u : ((uint32_t)(c >> 16 & 0xffff) < n ? 2u : ((uint32_t)(c & 0xffff) < n ? 1u : 0u))) << bit;
  }
  return most;
}

struct PickShared {
  double table[64];
  ull before, lds[2 * kWaves];
  uint32_t place, spots, at[kPartsMost + 1];
  uint32_t cut[2];
  union {
    LongWay far;
    List list;
    struct {
      uint32_t lane[kFewRoom];
      alignas(16) ull key[kFewRoom + 1];   // order_of and the index turned round: a larger one comes first
      ull sorted[kFewMost];
      alignas(16) ull idx[kFewMost + 1];
      double w[kFewMost];
      ull turn[2][kThreads];
    } few;
  };
};

// The largest t that n of the threads' keys reach, two bits a barrier
__device__ __forceinline__ uint32_t reached_by(uint32_t key, uint32_t n, Group& grp) {
  const ull both = grp.reduce<kWaves, ull>((ull)key << 32 | ~key, [](ull a, ull b) { return a & b; });
  const uint32_t same = (uint32_t)(both >> 32) | (uint32_t)both;   // bits that all keys share
  int bit = same == ~0u ? 0 : 32 - __clz(~same);
  bit += bit & 1;
  uint32_t t = bit >= 32 ? 0 : (uint32_t)(both >> 32) >> bit << bit;
  for (bit -= 2; bit >= 0; bit -= 2) {
    const ull c1 = __popcll(__ballot(key >= (t | 1u << bit))), c2 = __popcll(__ballot(key >= (t | 2u << bit))),
              c3 = __popcll(__ballot(key >= (t | 3u << bit)));
    ull c = grp.of_waves<kWaves>(c1 | c2 << 16 | c3 << 32);
#pragma unroll
    for (int o = 1; o < kWaves; o <<= 1) c += from_lane(c, o);
    t |= ((uint32_t)(c >> 32) >= n ? 3u : ((uint32_t)(c >> 16 & 0xffff) >= n ? 2u : ((uint32_t)(c & 0xffff) >= n ? 1u : 0u))) << bit;
  }
  return t;
}

// True, on all threads, where the row has to go the long way.
template <typename E>
__device__ __forceinline__ bool pick(const SampleArgs& p, const Work& ws, const Settings& st, const Weights& weight, PickShared& sh,
                                     Group& grp, ull* sub_units) {
  const int tid = threadIdx.x, row = ws.row0 + blockIdx.x, r = blockIdx.x, V = p.vocab;
  const Part* parts = ws.part + (int64_t)r * ws.parts;
  const Row<E> x(p, row);
  constexpr int LOW = kLow<E>;

  if (st.kind == kFew) {
    // At least top_k threads hold a token as large as the top_k-th largest of what
    // each holds at most, so the row's first top_k are among the tokens that are as
    // large: those of a little over top_k lanes, 16 each, and a few more than top_k of these.
    const int lanes = ws.subs * 64;
    const float* most = ws.most + (int64_t)r * lanes;
    constexpr int kStep = 10;   // loads on their way; kept, for rows of up to 163840
    float m[kStep], mine_most = -INFINITY;
    for (int i0 = (lanes - 1) / (kStep * kThreads) * (kStep * kThreads); i0 >= 0; i0 -= kStep * kThreads) {
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        const int i = i0 + k * kThreads + tid;
        m[k] = i < lanes ? most[i] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < kStep; ++k) mine_most = fmaxf(mine_most, m[k]);
    }
    const uint32_t mine_key = order_of(mine_most) >> LOW;
    const uint32_t least = reached_by(mine_key, st.top_k, grp);
    if (mine_key >= least) {
      auto take = [&](int i, float v) {
        if (const uint32_t k = order_of(v); k >> LOW >= least && k > kNone)
          if (const uint32_t at = atomicAdd(&sh.spots, 1u); at < kFewRoom) sh.few.lane[at] = i;
      };
#pragma unroll
      for (int k = 0; k < kStep; ++k) take(k * kThreads + tid, m[k]);
      for (int i = kStep * kThreads + tid; i < lanes; i += kThreads) take(i, most[i]);
    }
    __syncthreads();
    const uint32_t n = sh.spots;
    for (uint32_t i = tid; i < min(n, (uint32_t)kFewRoom) * 16; i += kThreads) {
      const int lane = sh.few.lane[i / 16], at = lane / 64 * kSub + x.at(i % 16, lane % 64);
      const uint32_t k = order_of(at < V ? (float)x.x[at] : -INFINITY);
      if (k >> LOW >= least && k > kNone)
        if (const uint32_t to = atomicAdd(&sh.place, 1u); to < kFewRoom) sh.few.key[to] = (ull)k << 32 | (uint32_t)~at;
    }
    __syncthreads();
    const uint32_t held = sh.place;
    if (n > kFewRoom || held > kFewRoom) return true;
    // the first top_k of them in their order
    const uint32_t k = min((uint32_t)st.top_k, held);
    if (tid == 0) sh.few.key[held] = 0;
    __syncthreads();
    ull own = tid < (int)held ? sh.few.key[tid] : 0;
    const bool sorts = held > kRanked;
    if (sorts) {
      own = held <= 512 ? in_order<512>(own, sh.few.turn) : in_order<1024>(own, sh.few.turn);
    } else {
      if (tid < (int)held) {
        const uint32_t rank = rank_of(own, sh.few.key, held);
        if (rank < k) sh.few.sorted[rank] = own;
      }
      __syncthreads();
      own = tid < (int)k ? sh.few.sorted[tid] : 0;
    }
    double w = 0;
    uint32_t idx = 0;
    if (tid < (int)k) {
      const ull mine = own;
      idx = ~(uint32_t)mine;
      w = weight(value_of((uint32_t)(mine >> 32)));
      sh.few.idx[tid] = ~idx;   // larger for the first
    }
    if (tid == (int)k) sh.few.idx[k] = 0;
    double sum;
    const double before = grp.scan<kWaves, double>(w, sum) - w;
    if (st.top_p < 1.0 && tid > 0 && !(before < st.top_p * sum)) w = 0;
    if (w < st.min_p) w = 0;
    // now by index
    if (sorts) {
      if (tid < (int)k) sh.few.w[tid] = w;
      const ull to = in_order<512>(tid < (int)k ? (ull)~idx << 32 | tid : 0, sh.few.turn);
      w = tid < (int)k ? sh.few.w[(uint32_t)to] : 0;
      if (tid < (int)k) sh.few.key[tid] = ~(uint32_t)(to >> 32);
    } else {
      if (tid < (int)k) {
        const uint32_t rank = rank_of((uint32_t)~idx, sh.few.idx, k);
        sh.few.w[rank] = w;
        sh.few.key[rank] = idx;
      }
      __syncthreads();
      w = tid < (int)k ? sh.few.w[tid] : 0;
    }
    const ull units = whole_of_list(w);
    ull total;
    const ull upto = grp.scan<kWaves, ull>(units, total), aim = share_of(st.u, total);
    if (upto > aim && upto - units <= aim) tell(p, row, (int)sh.few.key[tid], log(w / ((double)total * kListUnit)));
    return false;
  }

  // ---- the cuts: tokens stay whose key is over `key`, or just it with an index up to `idx` ----
  struct Cut {
    uint32_t key, idx;
    __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return (k > key) | ((k == key) & (i <= idx)); }
  } by_k{0, ~0u}, by_p{0, ~0u};
  Bounds b{-INFINITY, -INFINITY, -INFINITY, -INFINITY, 0, 0};
  uint32_t held = 0;
  double over_k = 0, over_p = 0;
  uint32_t over_n = 0;
  if (st.kind == kGrid) {
    b = ws.bounds[r];
    const int l = tid & 63;
    const bool mine = l < ws.parts;
    const uint32_t listed = mine ? parts[l].listed : 0;
    double ok = mine ? parts[l].over_k : 0, op = mine ? parts[l].over_p : 0;
    uint32_t on = mine ? parts[l].over_n : 0, upto = listed;
#pragma unroll
    for (int o = 1; o < kPartsMost; o <<= 1) {
      ok += __shfl_xor(ok, o);
      op += __shfl_xor(op, o);
      on += __shfl_xor(on, o);
      const uint32_t t = __shfl_up(upto, o);
      if (l >= o) upto += t;
    }
    over_k = __shfl(ok, 0);
    over_p = __shfl(op, 0);
    over_n = __shfl(on, 0);
    held = __shfl(upto, kPartsMost - 1);
    if (__any(listed > (uint32_t)ws.places)) return true;
    if (tid < kPartsMost) sh.at[tid + 1] = upto;
    if (tid == 0) sh.at[0] = 0;
    __syncthreads();
    for (uint32_t e = tid; e < held; e += kThreads) {
      int i = 0;
#pragma unroll
      for (int k = 1; k < kPartsMost; ++k) i += e >= sh.at[k];
      const uint32_t idx = ws.list[((int64_t)r * ws.parts + i) * ws.places + e - sh.at[i]];
      const float v = (float)x.x[idx];
      sh.list.key[e] = order_of(v) >> LOW;
      sh.list.idx[e] = idx;
      sh.list.units[e] = whole_of_list(weight(v));
    }
  }
  const bool cut_k = b.cut_k, cut_p = b.cut_p;
  auto value = [&](uint32_t key) { return value_of(key << LOW | (key >> (31 - LOW) & 1 ? 0 : (1u << LOW) - 1)); };
  auto of_k = [&](int i) {
    const float v = value(sh.list.key[i]);
    return cut_k && v >= b.k_lo && v < b.k_hi;
  };
  auto of_p = [&](int i) {
    const float v = value(sh.list.key[i]);
    return cut_p && v >= b.p_lo && v < b.p_hi;
  };
  __syncthreads();
  // Whether the cut of top_k is among the listed, and how much weight stays by it:
  // what must hold for the eight waves to go on is the same for all threads.
  const uint32_t* const key = sh.list.key;
  const uint32_t* const index = sh.list.idx;
  if (cut_k || cut_p) {
    // tokens of the window of top_k; the weights of both.  With all or nothing of the
    // former in the sum that top_p takes its share of, the aim lies between these two.
    ull n = 0, in_k = 0, in_p = 0;
    for (int i = tid; i < (int)held; i += kThreads) {
      const ull units = sh.list.units[i];
      const bool k = of_k(i);
      n += k;
      in_k += k ? units : 0;
      in_p += of_p(i) ? units : 0;
    }
    if (cut_k) {
      n = grp.sum<kWaves, ull>(n);
      in_k = grp.sum<kWaves, ull>(in_k);
      if (!(over_n < (uint32_t)st.top_k && over_n + n >= (uint32_t)st.top_k)) return true;
    }
    if (cut_p) {
      in_p = grp.sum<kWaves, ull>(in_p);
      const double lo = st.top_p * over_k, hi = st.top_p * (over_k + kListUnit * (double)in_k);
      // a window that ends with the tokens that top_k may leave needs no lower end of its own
      if (!((over_p < lo || over_p == 0) && (over_p + kListUnit * (double)in_p >= hi || (cut_k && b.p_lo <= b.k_lo)))) return true;
    }
  }
  if (tid >= kNearThreads) return false;

  if ((cut_k || cut_p) && held < kNearThreads) {
    // in their order, one to a thread: what stays is a first part of them
    ull *const all = sh.list.units + 1024, *const order = all + 1024, *const units = order + 1024;
    const ull mine = tid < (int)held ? (ull)key[tid] << 32 | (uint32_t)~index[tid] : 0;
    all[tid] = mine;   // and at least one zero
    if (tid == 0) sh.cut[0] = ~0u, sh.cut[1] = 0;   // none
    __syncthreads();
    if (tid < (int)held) {
      const uint32_t rank = rank_of(mine, all, held);
      order[rank] = mine;
      units[rank] = sh.list.units[tid];
    }
    __syncthreads();
    const ull own = tid < (int)held ? order[tid] : 0, unit = tid < (int)held ? units[tid] : 0;
    const float v = value((uint32_t)(own >> 32));
    const bool in_k = own && cut_k && v >= b.k_lo && v < b.k_hi, in_p = own && cut_p && v >= b.p_lo && v < b.p_hi;
    bool stay = own != 0;
    double sum = over_k;
    if (cut_k) {
      uint32_t n;
      const uint32_t at = grp.scan<kNear, uint32_t>(in_k, n);
      const bool first = in_k && at <= st.top_k - over_n;
      sum += kListUnit * (double)grp.sum<kNear, ull>(first ? unit : 0);
      stay &= first || v >= b.k_hi;
    }
    if (cut_p) {
      ull n;
      const ull at = grp.scan<kNear, ull>(in_p ? unit : 0, n);
      stay &= in_p && over_p + kListUnit * (double)(at - unit) < fmax(st.top_p * sum, 0x1p-1000);   // the first token stays
    }
    const uint32_t n = grp.sum_of_waves<kNear>(__popcll(__ballot(stay)));
    if (tid == (int)n - 1) {
      sh.cut[0] = (uint32_t)(own >> 32);
      sh.cut[1] = ~(uint32_t)own;
    }
    __syncthreads();
    by_k = {sh.cut[0], sh.cut[1]};
  } else if (cut_k || cut_p) {
    // the keys' common head
    uint32_t ones = ~0u, zeros = ~0u;
    for (int i = tid; i < (int)held; i += kNearThreads) ones &= key[i], zeros &= ~key[i];
    const ull both = grp.reduce<kNear, ull>((ull)ones << 32 | zeros, [](ull a, ull b) { return a & b; });
    const uint32_t same = (uint32_t)(both >> 32) | (uint32_t)both;
    const int bits = same == ~0u ? 0 : 32 - __clz(~same);
    const uint32_t head = bits == 32 ? 0 : (uint32_t)(both >> 32) >> bits << bits;
    double sum = over_k;
    if (cut_k) {
      const uint32_t n = st.top_k - over_n;
      by_k.key = nth_key(held, n, head, bits, key, grp, of_k);
      const uint32_t over = number_of(held, grp, [&](int i) { return key[i] > by_k.key && of_k(i); });
      auto tie = [&](int i) { return key[i] == by_k.key; };
      if (number_of(held, grp, tie) > n - over) by_k.idx = nth_index(held, n - over, V, index, grp, tie);
      ull mine = 0;
      for (int i = tid; i < (int)held; i += kNearThreads)
        if (of_k(i) && by_k.keeps(key[i], index[i])) mine += sh.list.units[i];
      sum += kListUnit * (double)grp.sum<kNear, ull>(mine);
    }
    if (cut_p) {
      const double aim = fmax(st.top_p * sum, 0x1p-1000);   // the first token stays
      auto over = [&](uint32_t t) {   // the weight before key t's tokens
        ull mine = 0;
        for (int i = tid; i < (int)held; i += kNearThreads)
          if (key[i] > t && of_p(i)) mine += sh.list.units[i];
        return over_p + kListUnit * (double)grp.sum<kNear, ull>(mine);
      };
      // the smallest key before which the aim is not reached: tokens of it stay
      uint32_t t = head | (bits == 32 ? ~0u : (1u << bits) - 1);
#pragma unroll 1
      for (int bit = bits - 1; bit >= 0; --bit)
        if (over(t & ~(1u << bit)) < aim) t &= ~(1u << bit);
      by_p.key = t;
      auto tie = [&](int i) { return key[i] == t; };
      const uint32_t ties = number_of(held, grp, tie);
      if (ties > 0) {
        const double n = fmax(ceil((aim - over(t)) / weight(value(t))), 1.0);
        if (n < (double)ties) by_p.idx = nth_index(held, (uint32_t)n, V, index, grp, tie);
      }
    }
  }
  // {0, ~0u}, what a cut that there is not keeps, is everything
  auto stays = [&](uint32_t k, uint32_t i) { return by_k.keeps(k, i) & by_p.keeps(k, i); };

  // ---- the sub ----
  const ull* sub = ws.sub + (int64_t)r * ws.subs;
  for (int s = tid; s < ws.subs; s += kNearThreads) sub_units[s] = sub[s];
  __syncthreads();
  const float sure = b.sure();
  const double one = ws.one;
  for (int i = tid; i < (int)held; i += kNearThreads)
    if (stays(key[i], index[i])) {
      const double w = weight(value(key[i]));
      if (w >= st.min_p) atomicAdd(&sub_units[index[i] / kSub], whole(w, one));
    }
  __syncthreads();
  const int per = (ws.subs + kNearThreads - 1) / kNearThreads, f0 = tid * per, f1 = min(f0 + per, ws.subs);
  ull mine = 0, total;
  for (int s = f0; s < f1; ++s) mine += sub_units[s];
  ull before = grp.scan<kNear, ull>(mine, total) - mine;
  const ull aim = share_of(st.u, total);
  if (before <= aim && before + mine > aim) {   // one thread
    int s = f0;
    for (; before + sub_units[s] <= aim; ++s) before += sub_units[s];
    sh.cut[0] = s;
    sh.before = before;
  }
  __syncthreads();
  const int s = (int)sh.cut[0];
  const ull left = aim - sh.before;

  // ---- the token: some in a row to a thread ----
  constexpr int kIn = kSub / kNearThreads;
  ull w[kIn], sums = 0;
  const int i0 = s * kSub + tid * kIn;
#pragma unroll
  for (int j = 0; j < kIn; ++j) {
    const int i = i0 + j;
    const float v = i < V ? (float)x.x[i] : -INFINITY;
    const double t = weight(v);
    // without branches: with them this compiler loses the zeros of all but the first
    w[j] = whole((t >= st.min_p) & ((v >= sure) | stays(order_of(v) >> LOW, i)) ? t : 0.0, one);
    sums += w[j];
  }
  ull all, upto = grp.scan<kNear, ull>(sums, all) - sums;
#pragma unroll
  for (int j = 0; j < kIn; ++j) {
    if (upto <= left && upto + w[j] > left) tell(p, row, i0 + j, log(weight((float)x.x[i0 + j]) / ((double)total * (one * 0x1p-52))));
    upto += w[j];
  }
  return false;
}

template <typename E> __global__ __launch_bounds__(kThreads, 8) void sample_pick_kernel(SampleArgs p, Work ws) {
  __shared__ PickShared sh;
  extern __shared__ ull sub_units[];   // [subs]
  const int tid = threadIdx.x, row = ws.row0 + blockIdx.x;
  const Settings st = settings_of(p, row, ws.few);
  const Part* parts = ws.part + (int64_t)blockIdx.x * ws.parts;
  const float M = top_of(parts, ws.parts);
  if (M == -INFINITY) {
    if (tid == 0) tell(p, row, -1, -INFINITY);
    return;
  }
  if (st.kind == kGreedy) {
    const uint64_t of = __ballot((tid & 63) < ws.parts && parts[(tid & 63) < ws.parts ? tid & 63 : 0].top == M);
    if (tid == 0) tell(p, row, (int)parts[__builtin_ctzll(of)].first, 0);
    return;
  }
  fill_table(sh.table);
  if (tid == 0) sh.place = sh.spots = 0;
  __syncthreads();
  const Weights weight{sh.table, steps_of(st.inv_t), M};
  Group grp{sh.lds};
  if ((M == INFINITY && st.kind != kFew) || pick<E>(p, ws, st, weight, sh, grp, sub_units)) {
    __syncthreads();
    long_way<E>(p, row, st, weight, ws.one, sh.far, grp);
  }
}

// ---- launches ----
constexpr int kEnough = 2;
// Parts of a row: enough workgroups for kEnough to a CU, of 16 subs at least (one to a
// wave), 2^18 tokens at most; of a few numbers the one whose waves have most even work.
struct Plan {
  int parts, subs, part_subs, places, few;
  int64_t rows;   // of a launch
  bool grid, gather;   // some row may need it
  size_t part_at, bounds_at, sub_at, most_at, list_at, cells_at, bytes;
};
Plan plan_of(const SampleArgs& a, int num_cus) {
  Plan pl;
  pl.subs = (a.vocab + kSub - 1) / kSub;
  pl.rows = std::min<int64_t>(a.rows, 1024);
  const int most = std::min(kPartsMost, (pl.subs + kWaves - 1) / kWaves);
  const int want = (int)std::max<int64_t>(1, std::min<int64_t>((kEnough * (int64_t)num_cus + pl.rows - 1) / pl.rows, most));
  pl.parts = want;
  auto rounds = [&](int parts) { return ((pl.subs + parts - 1) / parts + kWaves - 1) / kWaves; };
  for (int n = want + 1; n <= std::min(most, want + 3); ++n)
    if (n * rounds(n) < pl.parts * rounds(pl.parts)) pl.parts = n;
  pl.parts = std::max(pl.parts, (int)(((int64_t)a.vocab + (1 << 18) - 1) >> 18));
  pl.part_subs = (pl.subs + pl.parts - 1) / pl.parts;
  pl.parts = (pl.subs + pl.part_subs - 1) / pl.part_subs;
  pl.places = kListRow / pl.parts;
  pl.few = std::min(kFewMost, 32 * pl.subs);
  const bool greedy = !a.temperatures && !(a.temperature > 0.f);
  const int k = a.top_k > 0 && a.top_k < a.vocab ? a.top_k : a.vocab;                          // as settings_of takes it
  const bool cuts = a.top_ks || (k > pl.few && k < a.vocab);                                   // by number, with a grid
  pl.gather = !greedy && (a.top_ks || k > pl.few);
  pl.grid = (!greedy && cuts) || (pl.gather && (a.top_ps || a.top_p < 1.f));
  const bool some = !greedy && (a.top_ks || (k > 1 && k <= pl.few));                           // kFew
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t was = at;
    at += (n + 255) / 256 * 256;
    return was;
  };
  const size_t rp = (size_t)pl.rows * pl.parts;
  pl.part_at = take(rp * sizeof(Part));
  pl.bounds_at = take(pl.rows * sizeof(Bounds));
  pl.sub_at = take((size_t)pl.rows * pl.subs * sizeof(ull));
  pl.most_at = take(some ? (size_t)pl.rows * pl.subs * 64 * sizeof(float) : 0);
  pl.list_at = take(pl.gather ? rp * pl.places * sizeof(uint32_t) : 0);
  pl.cells_at = take(pl.grid ? rp * kCells * sizeof(uint32_t) : 0);
  pl.bytes = at;
  return pl;
}

template <typename E> hipError_t launch(const SampleArgs& a, const Plan& pl, char* ws, hipStream_t s) {
  Work w;
  w.part = (Part*)(ws + pl.part_at);
  w.bounds = (Bounds*)(ws + pl.bounds_at);
  w.sub = (ull*)(ws + pl.sub_at);
  w.most = (float*)(ws + pl.most_at);
  w.list = (uint32_t*)(ws + pl.list_at);
  w.cells = (uint32_t*)(ws + pl.cells_at);
  w.parts = pl.parts;
  w.subs = pl.subs;
  w.part_subs = pl.part_subs;
  w.one = 256.0;
  while (a.vocab * (0x1p52 / w.one) > 0x1p62) w.one *= 2;
  w.places = pl.places;
  w.few = pl.few;
  for (int64_t row0 = 0; row0 < a.rows; row0 += pl.rows) {
    w.row0 = (int)row0;
    const int rows = (int)std::min<int64_t>(pl.rows, a.rows - row0);
    sample_scan_kernel<E><<<rows * pl.parts, kThreads, 0, s>>>(a, w);
    if (pl.grid) sample_bounds_kernel<<<rows, kThreads, 0, s>>>(a, w);
    if (pl.gather) sample_gather_kernel<E><<<rows * pl.parts, kThreads, 0, s>>>(a, w);
    sample_pick_kernel<E><<<rows, kThreads, pl.subs * sizeof(ull), s>>>(a, w);
  }
  return hipGetLastError();
}

}  // namespace

size_t sample_workspace(const SampleArgs& a, int num_cus) { return a.rows ? plan_of(a, num_cus).bytes : 0; }

hipError_t sample_launch(const SampleArgs& a, int num_cus, void* ws, hipStream_t s) {
  const Plan pl = plan_of(a, num_cus);
  if (a.dtype == MQ_SAMPLE_F32) return launch<float>(a, pl, (char*)ws, s);
  return a.dtype == MQ_SAMPLE_BF16 ? launch<__bf16>(a, pl, (char*)ws, s) : launch<_Float16>(a, pl, (char*)ws, s);
}

}  // namespace mq
