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
// therefore taken in 64 bits (to 4e-14 of themselves), and sums in 64 bits too:
// as whole multiples of 2^-44 wherever atomics or a list's order would change
// what is added to what.
//
// A row is dealt out to `parts` workgroups, a wave taking 1024 tokens at a time
// (a sub).  What a row needs follows from its settings, which the GPU alone may
// know (Kind); the launches are the same for all of them:
//   scan    of every part: its largest logit, and by kind its first token; the
//           tokens that may be among the row's first top_k; the subs' sums; or how
//           much weight and how many tokens each cell of a grid over the
//           logits has.  Sums are relative to the part's own largest logit.
//   gather  where the grid was filled, or min_p alone cuts: the cells in which the
//           cuts fall, from all parts' grids; the subs' sums of what lies over
//           them, and a list of the tokens in them.
//   pick    the cuts among the listed tokens, the sub in which the running sum
//           passes its aim, and the token in it.
// A list that is too short (masses of equal logits at a cut) sends its row to
// the long way: cuts found digit by digit by one workgroup, pass after pass.
#include "mq_device.hpp"
#include "mq_sample.hpp"

#include "../../include/metal_native_amd.h"

#include <algorithm>

namespace mq {
namespace {

typedef unsigned long long ull;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kSub = 1024;
constexpr int kListRow = 8192;              // list entries of a row, over all parts
constexpr int kHeld = kListRow / kThreads;  // of them in a thread
constexpr int kFewMost = 512;               // top_k up to which a row may be Few

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

enum Kind { kGreedy, kFew, kGrid, kFloor, kAll };

struct Settings {
  double inv_t, top_p, min_p;
  int top_k;   // vocab: none
  float u;
  int kind;
};
// few: the largest top_k that goes by the parts' first tokens
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
           : s.top_k < p.vocab || s.top_p < 1.0 ? kGrid : (s.min_p > 0 ? kFloor : kAll);
  return s;
}

// ---- weights ----
// w = 2^(t / 64), t = (x - M) 64 log2(e) / T: the nearest whole number of t by
// a table and the exponent's bits, the rest by its series to the fourth power,
// (log(2) / 128)^5 / 120 = 4e-14 of w.  About 20 instructions where the library's exp takes
// twice as many.  0 for NaN and -inf, and under 2^-1020.
struct Weights {
  const double* table;   // 2^(i / 64)
  double c;
  float M;
  __device__ __forceinline__ double operator()(float x) const {
    const double d = x == M ? 0.0 : (double)x - (double)M, t = d * c;
    constexpr double kWhole = 0x1.8p52, kLn = 0.69314718055994530942 / 64;
    const double n = t + kWhole, f = (t - (n - kWhole)) * kLn;
    const int i = (int)(uint32_t)__double_as_longlong(n);
    double e = __builtin_fma(f, 1.0 / 24, 1.0 / 6);
    e = __builtin_fma(f, e, 0.5);
    e = __builtin_fma(f, e, 1.0) * f;
    const double w = table[i & 63];
    const long long bits = __double_as_longlong(__builtin_fma(w, e, w)) + ((long long)(i >> 6) << 52);
    return t >= -65280.0 ? __longlong_as_double(bits) : 0.0;
  }
};
__device__ __forceinline__ double steps_of(double inv_t) { return inv_t * (64 * 1.44269504088896340736); }
__device__ __forceinline__ void fill_table(double* table) {   // before a barrier
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(threadIdx.x / 64.0);
}
// w in 2^-44, to the nearest
__device__ __forceinline__ ull whole(double w) { return (ull)__double_as_longlong(w + 256.0) & ((1ull << 52) - 1); }
constexpr double kUnit = 0x1p-44;
// of a list's tokens, no more than kListRow of them, in 2^-50
__device__ __forceinline__ ull whole_of_list(double w) { return (ull)__double_as_longlong(w + 4.0) & ((1ull << 52) - 1); }
constexpr double kListUnit = 0x1p-50;

// ---- the grid: cells of 1/64 of a factor of two in weight, the same ones for all
// parts of a row; 1536 under the largest logit's by themselves, the rest by
// sixteens, what lies under all of these in the last one ----
constexpr int kFine = 1536, kCoarse = 512, kCells = kFine + kCoarse;
__device__ __forceinline__ float grid_scale(double inv_t) { return (float)fmin(steps_of(inv_t), 1e30); }
__device__ __forceinline__ int grid_of(float x, float scale) {   // grows with x
  const float g = fminf(fmaxf(floorf(x * scale), -0x1p29f), 0x1p29f);
  return x == INFINITY ? 1 << 29 : (int)g;
}
__device__ __forceinline__ int cell_of(int g, int top) {
  const int d = top - g;
  return d < kFine ? d : kFine + min(kCoarse - 1, (top >> 4) - (g >> 4));
}

// ---- a workgroup's sums ----
template <typename V, typename F> __device__ __forceinline__ V reduce(V v, V* lds, F&& f) {   // on every thread
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o; o >>= 1) v = f(v, (V)__shfl_xor(v, o));
  __syncthreads();
  if (lane == 0) lds[w] = v;
  __syncthreads();
  v = lds[0];
  for (int i = 1; i < kWaves; ++i) v = f(v, lds[i]);
  return v;
}
template <typename V> __device__ __forceinline__ V add_up(V v, V* lds) {
  return reduce<V>(v, lds, [](V a, V b) { return a + b; });
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
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) before += lds[i];
    all += lds[i];
  }
  return v + before;
}
// of 32-bit counts that are the same on a wave's lanes; one barrier, by turns in two halves of lds
__device__ __forceinline__ uint32_t count_up(uint32_t n, uint32_t* lds, int& turn) {
  turn ^= kWaves;
  if ((threadIdx.x & 63) == 0) lds[turn + (threadIdx.x >> 6)] = n;
  __syncthreads();
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) s += lds[turn + i];
  return s;
}

// ---- a wave's 1024 tokens ----
template <typename E> struct Row {
  const E* x;
  int V;
  bool aligned;   // its first element to 16 bytes
  __device__ __forceinline__ Row(const SampleArgs& p, int row) : x((const E*)p.logits + (int64_t)row * p.ld), V(p.vocab), aligned(((uintptr_t)x & 15) == 0) {}
  static constexpr int kPer = 16 / sizeof(E);
  // the lane's j-th: index within the sub, growing with j
  __device__ __forceinline__ int at(int j) const {
    const int lane = threadIdx.x & 63;
    return aligned ? j / kPer * (64 * kPer) + lane * kPer + j % kPer : j * 64 + lane;
  }
  __device__ __forceinline__ void load(int sub, float (&v)[16]) const {   // -inf past the row
    const int base = sub * kSub, lane = threadIdx.x & 63;
    if (aligned && base + kSub <= V) {
      typedef E vec __attribute__((ext_vector_type(kPer)));
      vec t[16 / kPer];
#pragma unroll
      for (int i = 0; i < 16 / kPer; ++i) t[i] = *(const vec*)(x + base + (i * 64 + lane) * kPer);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = (float)t[j / kPer][j % kPer];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = base + at(j);
        v[j] = i < V ? (float)x[i] : -INFINITY;
      }
    }
  }
};

// ---- what the launches hand on ----
struct Part {
  float top;       // largest logit
  uint32_t listed; // tokens that asked for a place in the list; past its length: it is not whole
  uint32_t first;  // kGreedy: the first token of that logit
  uint32_t pad;
  double tail;     // kGrid: weights that are in no cell
};
struct RowCut {   // by gather, for pick
  int cell_k, cell_p0, cell_p1;   // the cut of top_k falls in cell_k, that of top_p in cell_p0 .. cell_p1 (kCells: there is none)
  uint32_t before_n;              // tokens before cell_k
  double before_k, before_p;      // weight before cell_k, cell_p0
  double sum;                     // of all tokens
};
struct Work {
  Part* part;       // [rows, parts]
  RowCut* cut;      // [rows]
  double* sub;      // [rows, subs]
  uint32_t* list;   // [rows, parts, places]
  ull* weight;      // [rows, parts, kCells]
  uint32_t* number; // [rows, parts, kCells]
  int row0, parts, subs, places, few;
  __device__ __forceinline__ int first_sub(int part) const { return (int)((int64_t)subs * part / parts); }
};

template <typename E> __global__ __launch_bounds__(kThreads) void sample_scan_kernel(SampleArgs p, Work ws) {
  __shared__ double table[64];
  __shared__ union {
    ull weight[kCells];
    ull red[kWaves];
    uint32_t count[2 * kWaves];
  } sh;
  __shared__ uint32_t number[kCells], places;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = blockIdx.x / ws.parts, part = blockIdx.x - r * ws.parts, row = ws.row0 + r;
  const Settings st = settings_of(p, row, ws.few);
  const Row<E> x(p, row);
  const int s0 = ws.first_sub(part) + w, s1 = ws.first_sub(part + 1);
  fill_table(table);
  if (tid == 0) places = 0;
  float v[16], mine = -INFINITY;
  for (int s = s0; s < s1; s += kWaves) {
    x.load(s, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) mine = fmaxf(mine, v[j]);   // the number of the two, where one is NaN
  }
  const float M = __uint_as_float((uint32_t)reduce<ull>(__float_as_uint(mine), sh.red, [](ull a, ull b) {
    return (ull)__float_as_uint(fmaxf(__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)b)));
  }));
  Part& out = ws.part[(int64_t)r * ws.parts + part];
  if (tid == 0) out.top = M;
  __syncthreads();   // sh.red is read
  if (M == -INFINITY) {
    if (tid == 0) out.listed = 0;
    return;
  }
  const Weights weight{table, steps_of(st.inv_t), M};
  double* sub = ws.sub + (int64_t)r * ws.subs;
  if (st.kind == kGreedy) {
    uint32_t first = ~0u;
    for (int s = s0; s < s1 && first == ~0u; s += kWaves) {
      x.load(s, v);
#pragma unroll
      for (int j = 15; j >= 0; --j) first = v[j] == M ? s * kSub + x.at(j) : first;
    }
    first = (uint32_t)reduce<ull>(first, sh.red, [](ull a, ull b) { return a < b ? a : b; });
    if (tid == 0) out.first = first;
  } else if (st.kind == kAll) {
    for (int s = s0; s < s1; s += kWaves) {
      x.load(s, v);
      double sum = 0;
#pragma unroll 4
      for (int j = 0; j < 16; ++j) sum += weight(v[j]);
#pragma unroll
      for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
      if (lane == 0) sub[s] = sum;
    }
  } else if (st.kind == kFew) {
    // At least top_k of the threads hold a token as large as the top_k-th
    // largest of what each holds at most, so all of the row's first top_k in
    // this part are as large; about top_k tokens are, while it is half the threads or less.
    const uint32_t key = order_of(mine) >> kLow<E>;
    uint32_t least = 0;
    int turn = 0;
#pragma unroll 1
    for (int bit = 31 - kLow<E>; bit >= 0; --bit) {
      const uint32_t t = least | 1u << bit;
      if (count_up(__popcll(__ballot(key >= t)), sh.count, turn) >= (uint32_t)st.top_k) least = t;
    }
    uint32_t* list = ws.list + ((int64_t)r * ws.parts + part) * ws.places;
    const float low = value_of(least << kLow<E> | ((least >> (31 - kLow<E>)) & 1 ? 0 : (1u << kLow<E>) - 1));
    for (int s = s0; s < s1; s += kWaves) {
      x.load(s, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool take = v[j] >= low && v[j] > -INFINITY;
        const uint64_t all = __ballot(take);
        if (!all) continue;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&places, (uint32_t)__popcll(all));
        at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((1ull << lane) - 1));
        if (take && at < (uint32_t)ws.places) list[at] = s * kSub + x.at(j);
      }
    }
    __syncthreads();
    if (tid == 0) out.listed = places;
  } else if (st.kind == kGrid) {
    const bool count = st.top_k < p.vocab;
    const float scale = grid_scale(st.inv_t);
    const int top = grid_of(M, scale);
    // Of tokens under (1 - top_p) / 2 V of the part's largest weight, all of them
    // together are less than the cut leaves out: where nothing counts them they
    // need no cell
    const double least = count ? -1.0 : (1.0 - st.top_p) / (2.0 * p.vocab);
    for (int i = tid; i < kCells; i += kThreads) sh.weight[i] = 0, number[i] = 0;
    __syncthreads();
    double tail = 0;
    for (int s = s0; s < s1; s += kWaves) {
      x.load(s, v);
#pragma unroll 4
      for (int j = 0; j < 16; ++j) {
        const double wt = weight(v[j]);
        if (wt < least) {
          tail += wt;
        } else if (v[j] > -INFINITY) {
          const int cell = cell_of(grid_of(v[j], scale), top);
          atomicAdd(&sh.weight[cell], whole(wt));
          if (count) atomicAdd(&number[cell], 1u);
        }
      }
    }
    __syncthreads();
    ull* weights = ws.weight + ((int64_t)r * ws.parts + part) * kCells;
    for (int i = tid; i < kCells; i += kThreads) weights[i] = sh.weight[i];
    if (count) {
      uint32_t* numbers = ws.number + ((int64_t)r * ws.parts + part) * kCells;
      for (int i = tid; i < kCells; i += kThreads) numbers[i] = number[i];
    }
    __syncthreads();
    tail = add_up<double>(tail, (double*)sh.red);
    if (tid == 0) out.tail = tail;
  }
}

// The row's largest logit, over its parts
__device__ __forceinline__ float top_of(const Part* part, int parts) {
  float M = -INFINITY;
  for (int i = 0; i < parts; ++i) M = fmaxf(M, part[i].top);
  return M;
}

// Grids are laid over each other: a cell of a part's grid is one of the row's.
template <typename E> __global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleArgs p, Work ws) {
  __shared__ double table[64], red[kWaves];
  __shared__ RowCut cut;
  __shared__ uint32_t places;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = blockIdx.x / ws.parts, part = blockIdx.x - r * ws.parts, row = ws.row0 + r;
  const Settings st = settings_of(p, row, ws.few);
  if (st.kind != kGrid && st.kind != kFloor) return;
  Part* parts = ws.part + (int64_t)r * ws.parts;
  const float M = top_of(parts, ws.parts);
  if (M == -INFINITY) return;
  fill_table(table);
  if (tid == 0) {
    places = 0;
    cut.cell_k = cut.cell_p0 = cut.cell_p1 = kCells;
    cut.before_n = 0;
    cut.before_k = cut.before_p = cut.sum = 0;
  }
  __syncthreads();
  const Weights weight{table, steps_of(st.inv_t), M};
  const bool count = st.top_k < p.vocab;
  const float scale = grid_scale(st.inv_t);
  const int top = grid_of(M, scale);
  if (st.kind == kGrid) {
    const int b0 = 2 * tid;   // the thread's two cells
    double wt[2] = {0, 0}, tail = 0;
    uint32_t n[2] = {0, 0};
    for (int i = 0; i < ws.parts; ++i) {
      const float m = parts[i].top;
      if (m == -INFINITY) continue;
      const double f = weight(m);
      if (!count) tail += f * parts[i].tail;
      const int mt = grid_of(m, scale);
      const ull* pw = ws.weight + ((int64_t)r * ws.parts + i) * kCells;
      const uint32_t* pn = ws.number + ((int64_t)r * ws.parts + i) * kCells;
      auto take = [&](int k, int c) {
        wt[k] += f * kUnit * (double)pw[c];
        if (count) n[k] += pn[c];
      };
      if (b0 < kFine) {
        const int l = b0 - (top - mt);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (l + k >= 0 && l + k < kFine) take(k, l + k);
      } else {
        for (int k = 0; k < 2; ++k) {
          const int c = b0 + k - kFine, cell = (top >> 4) - c;   // values g with g >> 4 == cell, for the last c also the ones under it
          const bool last = c == kCoarse - 1;
          const int from = max((mt >> 4) - cell, 0), to = last ? kCoarse - 1 : min((mt >> 4) - cell, kCoarse - 1);
          for (int q = from; q <= to; ++q) take(k, kFine + q);
          // its fine cells that are not the row's
          const int lo = max(max(mt - (cell * 16 + 15), mt - top + kFine), 0), hi = last ? kFine - 1 : min(mt - cell * 16, kFine - 1);
          for (int q = lo; q <= hi; ++q) take(k, q);
        }
      }
    }
    double all, sum0 = scan<double>(wt[0] + wt[1], red, all) - (wt[0] + wt[1]);   // before the first
    const double sums[3] = {sum0, sum0 + wt[0], sum0 + wt[0] + wt[1]};
    uint32_t alln = 0, num0 = 0;
    if (count) num0 = scan<uint32_t>(n[0] + n[1], (uint32_t*)red, alln) - n[0] - n[1];
    const uint32_t nums[3] = {num0, num0 + n[0], num0 + n[0] + n[1]};
    __syncthreads();
    if (count)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (nums[k] < (uint32_t)st.top_k && nums[k + 1] >= (uint32_t)st.top_k) {
          cut.cell_k = b0 + k;
          cut.before_n = nums[k];
          cut.before_k = sums[k];
          cut.sum = sums[k + 1];   // with all of the cell
        }
    __syncthreads();
    if (tid == 0 && cut.cell_k == kCells) cut.sum = all + tail;
    __syncthreads();
    if (st.top_p < 1.0) {
      // what top_p is taken of is known but for cell_k
      const double lo = cut.cell_k < kCells ? cut.before_k : cut.sum, hi = cut.sum;
      const double aim0 = fmax(st.top_p, 0.0) * lo * (1 - 1e-9), aim1 = fmax(st.top_p, 0.0) * hi * (1 + 1e-9);
      const int end = min(cut.cell_k, kCells - 1);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (b0 + k <= end && sums[k + 1] > sums[k]) {
          if (sums[k + 1] >= aim0) atomicMin(&cut.cell_p0, b0 + k);
          if (sums[k + 1] >= aim1) atomicMin(&cut.cell_p1, b0 + k);
        }
      __syncthreads();
      if (tid == 0) {
        cut.cell_p0 = min(cut.cell_p0, end);
        cut.cell_p1 = min(cut.cell_p1, end);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (b0 + k == cut.cell_p0) cut.before_p = sums[k];
      __syncthreads();
    }
    if (part == 0 && tid == 0) ws.cut[r] = cut;
  }
  const int cell_k = cut.cell_k, p0 = cut.cell_p0, p1 = cut.cell_p1, sure = min(cell_k, p0);
  const int past = max(sure - 1, max(cell_k < kCells ? cell_k : 0, p1 < kCells ? p1 : 0));   // the last cell that counts
  const Row<E> x(p, row);
  const int s0 = ws.first_sub(part) + w, s1 = ws.first_sub(part + 1);
  double* sub = ws.sub + (int64_t)r * ws.subs;
  uint32_t* list = ws.list + ((int64_t)r * ws.parts + part) * ws.places;
  float v[16];
  // weights under min_p, as logits, with a margin for the division by T
  const double span = (log(st.min_p) - 1e-9) / st.inv_t;
  const double low = st.min_p > 0 ? (double)M + span - 1e-9 * fabs(span) : -INFINITY;
  for (int s = s0; s < s1; s += kWaves) {
    x.load(s, v);
    double sum = 0;
    if (st.kind == kFloor) {
#pragma unroll 4
      for (int j = 0; j < 16; ++j)
        if (v[j] == M || (double)v[j] >= low) {
          const double wt = weight(v[j]);
          sum += wt >= st.min_p ? wt : 0.0;
        }
    } else {
#pragma unroll 4
      for (int j = 0; j < 16; ++j) {
        const int cell = v[j] > -INFINITY ? cell_of(grid_of(v[j], scale), top) : kCells;
        if (!__any(cell <= past)) continue;
        if (cell < sure) {
          const double wt = weight(v[j]);
          sum += wt >= st.min_p ? wt : 0.0;
        }
        const bool take = cell < kCells && ((cell >= p0 && cell <= p1) || cell == cell_k);
        const uint64_t all = __ballot(take);
        if (all) {
          uint32_t at = 0;
          if (lane == 0) at = atomicAdd(&places, (uint32_t)__popcll(all));
          at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((1ull << lane) - 1));
          if (take && at < (uint32_t)ws.places) list[at] = s * kSub + x.at(j);
        }
      }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) sub[s] = sum;
  }
  __syncthreads();
  if (tid == 0) parts[part].listed = places;
}

struct LongWay {
  uint32_t cnt[2048];
  ull wt[2048], red[kWaves];
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
__device__ __noinline__ void long_way(const SampleArgs& p, int row, const Settings& st, const Weights& weigh, LongWay& sh) {
  uint32_t* const cnt = sh.cnt;
  ull *const wt = sh.wt, *const red = sh.red;
  auto& found = sh.found;
  const int tid = threadIdx.x, V = p.vocab;
  const E* x = (const E*)p.logits + (int64_t)row * p.ld;
  const int spare = max(14 - __clz(V), 0);   // sums of V weights below 2^63
  auto key = [&](int i) { return order_of((float)x[i]); };
  auto real = [&](uint32_t k) { return weigh(value_of(k)); };
  auto whole = [&](uint32_t k) { return mq::whole(real(k)) >> spare; };

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
  auto weight = [&](int i) {
    const uint32_t k = key(i);
    if (k <= kNone || (cut && (k < at || (k == at && i > last)))) return 0.0;
    const double w = real(k);
    return w >= st.min_p ? w : 0.0;
  };
  double sum = 0;
  for (int i = tid; i < V; i += kThreads) sum += weight(i);
  const double total = add_up<double>(sum, (double*)red), aim = (double)st.u * total;
  double before = 0;
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const double w = i < V ? weight(i) : 0;
    double all;
    const double r = scan<double>(w, (double*)red, all) + before;
    // what rounding leaves under the aim at the row's end goes to the last token
    const ull pick = w > 0 && r > aim ? (ull)i : ~0ull, best = reduce<ull>(pick, red, [](ull a, ull b) { return a < b ? a : b; });
    const ull back = reduce<ull>(w > 0 ? (ull)i + 1 : 0, red, [](ull a, ull b) { return a > b ? a : b; });
    if (back) sh.found.bin = (uint32_t)back - 1;
    if (best != ~0ull) {
      sh.found.bin = (uint32_t)best;
      break;
    }
    before += all;
  }
  __syncthreads();
  if (tid == 0) tell(p, row, (int)sh.found.bin, log(weigh((float)x[sh.found.bin]) / total));
}

// ---- the last launch: a workgroup for each row ----
struct Held {   // list entries in registers; key 0: none
  uint32_t key[kHeld], idx[kHeld];
};
// The n-th largest key of those that are true to `of`, as bits from kLow on, among
// `bits` of them under a common head; one barrier a bit
template <int LOW, typename F>
__device__ __forceinline__ uint32_t nth_key(const Held& h, uint32_t n, uint32_t head, int bits, uint32_t* lds, int& turn, F&& of) {
  uint32_t least = head;
#pragma unroll 1
  for (int bit = bits - 1; bit >= 0; --bit) {
    const uint32_t t = least | 1u << bit;
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) c += __popcll(__ballot(of(j) && h.key[j] >> LOW >= t));
    if (count_up(c, lds, turn) >= n) least = t;
  }
  return least;
}
// The n-th smallest index of those that are true to `of`
template <typename F>
__device__ __forceinline__ uint32_t nth_index(const Held& h, uint32_t n, int vocab, uint32_t* lds, int& turn, F&& of) {
  uint32_t most = 0;   // fewer than n lie under it
#pragma unroll 1
  for (int bit = 31 - __clz(vocab); bit >= 0; --bit) {
    const uint32_t t = most | 1u << bit;
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) c += __popcll(__ballot(of(j) && h.idx[j] < t));
    if (count_up(c, lds, turn) < n) most = t;
  }
  return most;
}
template <typename F> __device__ __forceinline__ uint32_t number_of(uint32_t* lds, int& turn, F&& of) {
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) c += __popcll(__ballot(of(j)));
  return count_up(c, lds, turn);
}

template <typename E> __global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs p, Work ws) {
  __shared__ double table[64], red[kWaves];
  __shared__ uint32_t count[2 * kWaves], place;
  __shared__ union {
    LongWay far;
    struct {
      ull key[kFewMost];   // order_of and the index turned round: a larger one comes first
      ull sorted[kFewMost];
      double w[kFewMost];
    } few;
    ull sub[4096 + 1];
  } sh;
  const int tid = threadIdx.x, row = ws.row0 + blockIdx.x, r = blockIdx.x, V = p.vocab;
  const Settings st = settings_of(p, row, ws.few);
  const Part* parts = ws.part + (int64_t)r * ws.parts;
  const float M = top_of(parts, ws.parts);
  if (M == -INFINITY) {
    if (tid == 0) tell(p, row, -1, -INFINITY);
    return;
  }
  if (st.kind == kGreedy) {
    if (tid == 0) {
      int i = 0;
      while (parts[i].top != M) ++i;
      tell(p, row, (int)parts[i].first, 0);
    }
    return;
  }
  fill_table(table);
  if (tid == 0) place = 0;
  __syncthreads();
  const Weights weight{table, steps_of(st.inv_t), M};
  const Row<E> x(p, row);
  constexpr int LOW = kLow<E>;
  int turn = 0;
  const double aim_share = (double)st.u;

  // ---- the listed tokens ----
  Held h;
  uint32_t held = 0;
  bool whole_list = true;
  if (st.kind == kFew || st.kind == kGrid) {
    for (int i = 0; i < ws.parts; ++i) {
      whole_list &= parts[i].listed <= (uint32_t)ws.places;
      held += parts[i].listed;
    }
    if (!whole_list) {
      long_way<E>(p, row, st, weight, sh.far);
      return;
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      uint32_t e = tid + j * kThreads;
      h.key[j] = h.idx[j] = 0;
      if (e < held) {
        int i = 0;
        while (e >= parts[i].listed) e -= parts[i++].listed;
        h.idx[j] = ws.list[((int64_t)r * ws.parts + i) * ws.places + e];
        h.key[j] = order_of((float)x.x[h.idx[j]]);
      }
    }
  }
  if (st.kind == kFew) {
    // the first top_k of the list, by its keys and where they are equal by index
    const uint32_t k = min((uint32_t)st.top_k, held);
    auto any = [&](int j) { return h.key[j] != 0; };
    const uint32_t at = nth_key<LOW>(h, k, 0, 32 - LOW, count, turn, any);
    const uint32_t over = number_of(count, turn, [&](int j) { return h.key[j] >> LOW > at; });
    auto tie = [&](int j) { return h.key[j] >> LOW == at && h.key[j] != 0; };
    const uint32_t ties = number_of(count, turn, tie);
    const uint32_t last = ties > k - over ? nth_index(h, k - over, V, count, turn, tie) : ~0u;
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (h.key[j] >> LOW > at || (tie(j) && h.idx[j] <= last))
        sh.few.key[atomicAdd(&place, 1u)] = (ull)h.key[j] << 32 | (uint32_t)~h.idx[j];
    __syncthreads();
    ull mine = 0;
    if (tid < (int)k) {
      mine = sh.few.key[tid];
      uint32_t rank = 0;
      for (uint32_t i = 0; i < k; ++i) rank += sh.few.key[i] > mine;
      sh.few.sorted[rank] = mine;
    }
    __syncthreads();
    double w = 0;
    uint32_t idx = 0;
    if (tid < (int)k) {
      mine = sh.few.sorted[tid];
      idx = ~(uint32_t)mine;
      w = weight(value_of((uint32_t)(mine >> 32)));
    }
    double sum;
    const double before = scan<double>(w, red, sum) - w;
    if (st.top_p < 1.0 && tid > 0 && !(before < st.top_p * sum)) w = 0;
    if (w < st.min_p) w = 0;
    if (tid < (int)k) sh.few.w[tid] = w;
    __syncthreads();
    double upto = 0, total = 0;
    if (tid < (int)k) {
      for (uint32_t i = 0; i < k; ++i) {
        const double t = sh.few.w[i];
        total += t;
        upto += ~(uint32_t)sh.few.sorted[i] <= idx ? t : 0.0;
      }
    }
    const bool hit = w > 0 && upto > aim_share * total;
    const ull first = reduce<ull>(hit ? (ull)idx << 32 | tid : ~0ull, (ull*)red, [](ull a, ull b) { return a < b ? a : b; });
    if (first != ~0ull ? tid == (int)(uint32_t)first : tid == 0) tell(p, row, (int)idx, log(w / total));
    return;
  }

  // ---- the cuts: tokens stay whose key is over `key`, or just it with an index up to `idx` ----
  struct Cut {
    uint32_t key, idx;
    __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
  } cut_k{0, ~0u}, cut_p{0, ~0u};
  RowCut rc{};
  const float scale = grid_scale(st.inv_t);
  const int top = grid_of(M, scale);
  int sure = kCells;
  auto cell = [&](uint32_t key) { return cell_of(grid_of(value_of(key), scale), top); };
  if (st.kind == kGrid) {
    rc = ws.cut[r];
    sure = min(rc.cell_k, rc.cell_p0);
    ull units[kHeld];
    bool of_k[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      units[j] = h.key[j] ? whole_of_list(weight(value_of(h.key[j]))) : 0;
      of_k[j] = h.key[j] && cell(h.key[j]) == rc.cell_k;
    }
    // the keys' common head
    uint32_t ones = ~0u, zeros = ~0u;
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (h.key[j]) ones &= h.key[j] >> LOW, zeros &= ~(h.key[j] >> LOW);
    const ull both = reduce<ull>((ull)ones << 32 | zeros, (ull*)red, [](ull a, ull b) { return a & b; });
    const uint32_t same = (uint32_t)(both >> 32) | (uint32_t)both;
    const int bits = same == ~0u ? 0 : 32 - __clz(~same);
    const uint32_t head = bits == 32 ? 0 : (uint32_t)(both >> 32) >> bits << bits;
    double sum = rc.sum;
    if (rc.cell_k < kCells) {
      const uint32_t n = st.top_k - rc.before_n;
      auto of = [&](int j) { return of_k[j]; };
      cut_k.key = nth_key<LOW>(h, n, head, bits, count, turn, of);
      const uint32_t over = number_of(count, turn, [&](int j) { return of_k[j] && h.key[j] >> LOW > cut_k.key; });
      auto tie = [&](int j) { return of_k[j] && h.key[j] >> LOW == cut_k.key; };
      if (number_of(count, turn, tie) > n - over) cut_k.idx = nth_index(h, n - over, V, count, turn, tie);
      ull mine = 0;
#pragma unroll
      for (int j = 0; j < kHeld; ++j) mine += of_k[j] && cut_k.keeps(h.key[j] >> LOW, h.idx[j]) ? units[j] : 0;
      sum = rc.before_k + kListUnit * (double)add_up<ull>(mine, (ull*)red);
    }
    if (rc.cell_p0 < kCells) {
      const double aim = fmax(st.top_p * sum, 0x1p-1000);   // the first token stays
      bool of_p[kHeld];
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        const int c = h.key[j] ? cell(h.key[j]) : -1;
        of_p[j] = c >= rc.cell_p0 && c <= rc.cell_p1;
      }
      auto over = [&](uint32_t t) {   // the weight before key t's tokens
        ull mine = 0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) mine += of_p[j] && h.key[j] >> LOW > t ? units[j] : 0;
        return rc.before_p + kListUnit * (double)add_up<ull>(mine, (ull*)red);
      };
      // the smallest key before which the aim is not reached: tokens of it stay
      uint32_t t = head | (bits == 32 ? ~0u : (1u << bits) - 1);
#pragma unroll 1
      for (int bit = bits - 1; bit >= 0; --bit)
        if (over(t & ~(1u << bit)) < aim) t &= ~(1u << bit);
      cut_p.key = t;
      auto tie = [&](int j) { return of_p[j] && h.key[j] >> LOW == t; };
      const uint32_t ties = number_of(count, turn, tie);
      if (ties > 0) {
        const double w = weight(value_of(t << LOW | (((t >> (31 - LOW)) & 1) ? 0 : (1u << LOW) - 1)));
        const double n = fmax(ceil((aim - over(t)) / w), 1.0);
        if (n < (double)ties) cut_p.idx = nth_index(h, (uint32_t)n, V, count, turn, tie);
      }
    }
  }
  auto stays = [&](float v, uint32_t i) {   // a token in no cell over the cuts
    const uint32_t k = order_of(v) >> LOW;
    return (rc.cell_k == kCells || st.kind != kGrid || cut_k.keeps(k, i)) && (rc.cell_p0 == kCells || st.kind != kGrid || cut_p.keeps(k, i));
  };

  // ---- the sub ----
  const double* sub = ws.sub + (int64_t)r * ws.subs;
  __syncthreads();
  for (int s = tid; s < ws.subs; s += kThreads) sh.sub[s] = 0;
  __syncthreads();
  if (st.kind == kGrid)
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (h.key[j] && stays(value_of(h.key[j]), h.idx[j])) {
        const double w = weight(value_of(h.key[j]));
        if (w >= st.min_p) atomicAdd(&sh.sub[h.idx[j] / kSub], whole_of_list(w));
      }
  __syncthreads();
  const int per = (ws.subs + kThreads - 1) / kThreads, f0 = tid * per;
  auto sum_of = [&](int s) {
    if (st.kind != kAll) return sub[s] + kListUnit * (double)sh.sub[s];
    int i = 0;
    while (s >= ws.first_sub(i + 1)) ++i;
    return parts[i].top == -INFINITY ? 0.0 : sub[s] * weight(parts[i].top);
  };
  double mine = 0;
  for (int s = f0; s < min(f0 + per, ws.subs); ++s) mine += sum_of(s);
  double total;
  double before = scan<double>(mine, red, total) - mine;
  const double aim = aim_share * total;
  ull found = ~0ull, back = 0;
  double found_before = 0, back_before = 0;
  for (int s = f0; s < min(f0 + per, ws.subs); ++s) {
    const double w = sum_of(s);
    if (w > 0) {
      back = s + 1;
      back_before = before;
      if (found == ~0ull && before + w > aim) {
        found = s;
        found_before = before;
      }
    }
    before += w;
  }
  const ull first = reduce<ull>(found, (ull*)red, [](ull a, ull b) { return a < b ? a : b; });
  const ull end = reduce<ull>(back, (ull*)red, [](ull a, ull b) { return a > b ? a : b; });
  const int s = first != ~0ull ? (int)first : (int)end - 1;   // rounding may leave the sum under its aim
  __syncthreads();
  if (first != ~0ull ? found == first : back == end) red[0] = first != ~0ull ? found_before : back_before;
  __syncthreads();
  const double left = aim - red[0];
  __syncthreads();

  // ---- the token ----
  const int i = s * kSub + tid;
  const float v = i < V ? (float)x.x[i] : -INFINITY;
  double w = weight(v);
  if (w < st.min_p) w = 0;
  if (st.kind == kGrid && w > 0 && cell_of(grid_of(v, scale), top) >= sure && !stays(v, i)) w = 0;
  double all;
  const double upto = scan<double>(w, red, all);
  const ull hit = reduce<ull>(w > 0 && upto > left ? (ull)tid : ~0ull, (ull*)red, [](ull a, ull b) { return a < b ? a : b; });
  const ull stop = reduce<ull>(w > 0 ? (ull)tid + 1 : 0, (ull*)red, [](ull a, ull b) { return a > b ? a : b; });
  if (tid == (hit != ~0ull ? (int)hit : (int)stop - 1)) tell(p, row, i, log(w / total));
}

// ---- launches ----
// Parts of a row: enough workgroups for four to a CU, of 16 subs at least (one to a wave), 2^18 tokens at most
struct Plan {
  int parts, subs, places, few;
  int64_t rows;   // of a launch
  bool gather;    // some row may need it
  size_t part_at, cut_at, sub_at, list_at, weight_at, number_at, bytes;
};
Plan plan_of(const SampleArgs& a, int num_cus) {
  Plan pl;
  pl.subs = (a.vocab + kSub - 1) / kSub;
  pl.rows = std::min<int64_t>(a.rows, 1024);
  const int64_t want = (4 * (int64_t)num_cus + pl.rows - 1) / std::max<int64_t>(pl.rows, 1);
  pl.parts = (int)std::max<int64_t>(1, std::min<int64_t>({want, 16, (pl.subs + kWaves - 1) / kWaves}));
  pl.parts = std::max(pl.parts, (int)(((int64_t)a.vocab + (1 << 18) - 1) >> 18));
  pl.places = kListRow / pl.parts;
  const int least = pl.subs / pl.parts;   // subs of the smallest part
  pl.few = std::min({kFewMost, 32 * std::min(least, kWaves), pl.places / 2});
  const bool greedy = !a.temperatures && !(a.temperature > 0.f);
  const bool cuts = a.top_ks || (a.top_k > pl.few && a.top_k < a.vocab);                       // by number, with a grid
  const bool shares = !(!a.top_ks && a.top_k >= 1 && a.top_k <= pl.few) && (a.top_ps || a.min_ps || a.top_p < 1.f || a.min_p > 0.f);
  pl.gather = !greedy && (cuts || shares);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t was = at;
    at += (n + 255) / 256 * 256;
    return was;
  };
  const size_t rp = (size_t)pl.rows * pl.parts;
  pl.part_at = take(rp * sizeof(Part));
  pl.cut_at = take(pl.rows * sizeof(RowCut));
  pl.sub_at = take((size_t)pl.rows * pl.subs * sizeof(double));
  pl.list_at = take(rp * pl.places * sizeof(uint32_t));
  pl.weight_at = take(pl.gather ? rp * kCells * sizeof(ull) : 0);
  pl.number_at = take(pl.gather ? rp * kCells * sizeof(uint32_t) : 0);
  pl.bytes = at;
  return pl;
}

template <typename E> hipError_t launch(const SampleArgs& a, const Plan& pl, char* ws, hipStream_t s) {
  Work w;
  w.part = (Part*)(ws + pl.part_at);
  w.cut = (RowCut*)(ws + pl.cut_at);
  w.sub = (double*)(ws + pl.sub_at);
  w.list = (uint32_t*)(ws + pl.list_at);
  w.weight = (ull*)(ws + pl.weight_at);
  w.number = (uint32_t*)(ws + pl.number_at);
  w.parts = pl.parts;
  w.subs = pl.subs;
  w.places = pl.places;
  w.few = pl.few;
  for (int64_t row0 = 0; row0 < a.rows; row0 += pl.rows) {
    w.row0 = (int)row0;
    const int rows = (int)std::min<int64_t>(pl.rows, a.rows - row0);
    sample_scan_kernel<E><<<rows * pl.parts, kThreads, 0, s>>>(a, w);
    if (pl.gather) sample_gather_kernel<E><<<rows * pl.parts, kThreads, 0, s>>>(a, w);
    sample_pick_kernel<E><<<rows, kThreads, 0, s>>>(a, w);
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
