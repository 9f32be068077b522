// The paged cache's own kernels: rotary positions with the new keys and values
// written into their pages, and eviction by accumulated attention weight.
// Both move memory and little else.
#include "mq_paged_dev.hpp"

#include <algorithm>

namespace mq {
namespace {

// ---- rotary positions ----
//
// Frequency f of a head turns the pair (x_f, x_{f + D/2}) by the angle of the
// axis that owns f: (x cos - y sin, y cos + x sin), products and their sum in
// fp32, one rounding.  A thread takes eight frequencies of one token and walks
// over heads with their cosines and sines in registers: one 16-byte load per
// half head, and the tables are read once per thread instead of once per head.
// Bound by memory: 5262 tokens of 28 heads over 4, bf16, three axes, 100 MB: 18.6 us
// (5.4 TB/s; a large copy 4.95), 22 with the launch; one token 3 us, the launch.
template <typename T> struct V8 { typedef typename T::e v __attribute__((ext_vector_type(8))); };
typedef float f8 __attribute__((ext_vector_type(8)));

template <typename T>
__global__ __launch_bounds__(256) void paged_rope_kernel(PagedRopeArgs p, int split, int chunks_log) {
  typedef typename V8<T>::v v8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)idx & ((1 << chunks_log) - 1);
  const int64_t rest = idx >> chunks_log;
  const int t = (int)(rest / split), first = (int)(rest % split);
  if (t >= p.rows) return;
  const int half = p.D / 2, f0 = 8 * c, heads = p.H + 2 * p.KVH;
  auto row_of = [&](int axis) {
    const int64_t x = p.pos[(int64_t)axis * p.ld_pos + t];
    return x < 0 ? 0 : (x < p.table_rows ? x : p.table_rows - 1);   // never past the tables
  };
  int axis = 0;
  while (axis < p.axes - 1 && f0 >= p.sec_end[axis]) ++axis;
  f8 cs, sn;
  if (f0 + 8 <= p.sec_end[axis]) {
    const int64_t x = row_of(axis);
    const f4* a = (const f4*)(p.cos_t + x * p.ld_cos + f0);
    const f4* b = (const f4*)(p.sin_t + x * p.ld_sin + f0);
    const f4 a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
    cs = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
    sn = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      while (axis < p.axes - 1 && f0 + e >= p.sec_end[axis]) ++axis;
      const int64_t x = row_of(axis);
      cs[e] = p.cos_t[x * p.ld_cos + f0 + e];
      sn[e] = p.sin_t[x * p.ld_sin + f0 + e];
    }
  }
  // the slot of the token's key and value, where the thread has such a head
  int page = -1, in = 0;
  if (first + (heads - 1 - first) / split * split >= p.H) {
    int s = t;
    if (p.cu) {   // the last sequence that starts at or before t
      int lo = 0, hi = p.b;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid] <= t) lo = mid;
        else hi = mid;
      }
      s = lo;
    }
    if (s < p.b) {
      const PagedSeq q = paged_seq(s, p.cu ? p.cu[s] : 0, p.cu ? p.cu[s + 1] : 0, p.cu != nullptr, p.lens[s], 0, p.rows,
                                   p.cap);
      const int j = q.len - q.n + (t - q.start);
      if (t >= q.start && t < q.start + q.n) page = paged_page(p.table + (int64_t)s * p.ld_table, j, q.len, p.shift, p.pages);
      in = j & ((1 << p.shift) - 1);
    }
  }
  const typename T::e* src = (const typename T::e*)p.qkv + (int64_t)t * p.ld_qkv + f0;
#pragma unroll 2
  for (int a = first; a < heads; a += split) {
    const v8 x = *(const v8*)(src + a * p.D), y = *(const v8*)(src + a * p.D + half);
    v8 u = x, v = y;
    if (a < p.H + p.KVH) {
      const f8 xf = __builtin_convertvector(x, f8), yf = __builtin_convertvector(y, f8);
      u = __builtin_convertvector(xf * cs - yf * sn, v8);
      v = __builtin_convertvector(yf * cs + xf * sn, v8);
    }
    typename T::e* dst = (typename T::e*)p.q_out + ((int64_t)t * p.H + a) * p.D;
    if (a >= p.H) {
      if (page < 0) continue;
      const bool key = a < p.H + p.KVH;
      const PagedCache& k = key ? p.k : p.v;
      dst = (typename T::e*)const_cast<void*>(k.ptr) + page * k.page + (a - p.H - (key ? 0 : p.KVH)) * k.head +
            (int64_t)in * k.slot;
    }
    *(v8*)(dst + f0) = u;
    *(v8*)(dst + f0 + half) = v;
  }
}

// ---- eviction ----
//
// Of a sequence's len slots and one key/value head the last `recent` stay and,
// of those before, the ones of largest weight that fill the budget (ties: the
// lowest slot), all in their order.  The smallest weight that stays is found
// digit by digit (11, 11 and 10 bits of an order-preserving integer) with
// histograms in LDS; a second look counts, a third lists the slots.  Each of a
// head's workgroups does this for itself (a head's weights are at most some
// hundred KiB, in L2) and then moves its own part of the slots: one launch and
// nothing passed between workgroups.
// Eight sequences of 20-32 thousand slots to 8192, 8 heads, 547 MB moved: 143 us
// (110 at the copy rate; the looks at up to 128 KiB of weights come before anything
// moves); 1100 slots to 512: 10.9 us.  Without all threads summing the histograms
// and weights kept in registers 212 and 21.7; with two workgroups per CU 159.
constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64, kEvictList = 2048;

__device__ __forceinline__ uint32_t order_key(float v) {   // NaN above all, -0 like +0
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct EvictShared {
  uint32_t hist[4][2048];
  int list[kEvictList];
  uint32_t count[32 * kEvictWaves];   // per 1024 slots and wave: above the threshold | equal to it << 16
  uint32_t wave_sum[kEvictWaves];
  uint32_t digit;
  int above, zeros;
};

// E: weights per thread, kept in registers from the first look to the last (a
// head of at most 1024 E slots); 0: any number, read again each time.
template <int E>
__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(PagedEvictArgs p, int parts, int per) {
  __shared__ EvictShared sh;
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
  const int part = blockIdx.x % parts, kv = (blockIdx.x / parts) % p.KVH, s = blockIdx.x / parts / p.KVH;
  int len = p.lens[s];
  len = len < 0 ? 0 : (len > p.cap ? p.cap : len);
  const int kept_n = len < p.budget ? len : p.budget;
  const int old = len - p.recent > 0 ? len - p.recent : 0;
  const int r_begin = part * per, r_end = min(r_begin + per, p.budget);
  const float* mass = p.mass + s * p.mass_b + kv * p.mass_h;
  const bool cut = len > p.budget;
  const int from_old = cut ? p.budget - (len - old) : 0;   // how many of the old slots stay

  if (cut && from_old > 0 && r_begin < from_old) {
    constexpr uint32_t kZero = 0x80000000u;
    constexpr int N = E > 0 ? E : 1;
    uint32_t key[N];
    if constexpr (E > 0) {
      float m[N];
#pragma unroll
      for (int i = 0; i < N; ++i) m[i] = tid + i * kEvictThreads < old ? mass[tid + i * kEvictThreads] : 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) key[i] = order_key(m[i]);
    }
    auto each = [&](auto&& f) {   // f(slot, key) of the thread's slots
      if constexpr (E > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (tid + i * kEvictThreads < old) f(tid + i * kEvictThreads, key[i]);
      } else {
#pragma unroll 4
        for (int j = tid; j < old; j += kEvictThreads) f(j, order_key(mass[j]));
      }
    };
    uint32_t prefix = 0, done = 0;   // digits found so far, and their bits
    int need = from_old;             // how many stay among the slots that match them
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass == 2 ? 10 : 11, shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      for (int i = tid; i < 4 * 2048 / 4; i += kEvictThreads) ((u4*)&sh.hist[0][0])[i] = (u4){0u, 0u, 0u, 0u};
      if (tid == 0) sh.zeros = 0;
      __syncthreads();
      int zeros = 0;
      // weights that are exactly zero are many: counted apart, not one by one in one histogram cell
      each([&](int, uint32_t k) {
        if (k == kZero) ++zeros;
        else if ((k & done) == prefix) atomicAdd(&sh.hist[w & 3][(k >> shift) & ((1u << bits) - 1)], 1u);
      });
      if ((kZero & done) == prefix) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) zeros += __shfl_xor(zeros, o);
        if (lane == 0 && zeros) atomicAdd(&sh.zeros, zeros);
      }
      __syncthreads();
      // thread t: cells top - 2 t and top - 2 t - 1, summed from the top
      const int top = (1 << bits) - 1 - 2 * tid, zc = (kZero >> shift) & ((1u << bits) - 1);
      int c0 = 0, c1 = 0;
      if (top > 0) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint2 h2v = *(const uint2*)&sh.hist[x][top - 1];
          c1 += h2v.x;
          c0 += h2v.y;
        }
        if (zc == top) c0 += sh.zeros;
        if (zc == top - 1) c1 += sh.zeros;
      }
      int sum = c0 + c1;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(sum, o);
        if (lane >= o) sum += x;
      }
      if (lane == 63) sh.wave_sum[w] = sum;
      __syncthreads();
      int before = sum - c0 - c1;
      for (int x = 0; x < w; ++x) before += sh.wave_sum[x];
      if (before < need && before + c0 + c1 >= need) {
        const bool first = before + c0 >= need;
        sh.digit = (uint32_t)(first ? top : top - 1);
        sh.above = first ? before : before + c0;
      }
      __syncthreads();
      prefix |= sh.digit << shift;
      done |= ((1u << bits) - 1) << shift;
      need -= sh.above;
      __syncthreads();
    }
    // stays: key > prefix, and the first `need` of key == prefix
    const uint64_t below = (1ull << lane) - 1;
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool in = tid + i * kEvictThreads < old;
        const uint64_t mg = __ballot(in && key[i] > prefix), me = __ballot(in && key[i] == prefix);
        if (lane == 0) sh.count[i * kEvictWaves + w] = (uint32_t)__popcll(mg) | (uint32_t)__popcll(me) << 16;
      }
      __syncthreads();
      if (w == 0) {   // sums of all before, in the slots' order (both fields at most 1024 E <= 32768)
        constexpr int C = N * kEvictWaves / 64 > 0 ? N * kEvictWaves / 64 : 1;
        uint32_t mine = 0;
        for (int x = 0; x < C; ++x) mine += lane * C + x < N * kEvictWaves ? sh.count[lane * C + x] : 0u;
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t x = __shfl_up(sum, o);
          if (lane >= o) sum += x;
        }
        uint32_t before = sum - mine;
        for (int x = 0; x < C; ++x)
          if (lane * C + x < N * kEvictWaves) {
            const uint32_t c = sh.count[lane * C + x];
            sh.count[lane * C + x] = before;
            before += c;
          }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = tid + i * kEvictThreads;
        const bool in = j < old, gt = in && key[i] > prefix, eq = in && key[i] == prefix;
        const uint64_t mg = __ballot(gt), me = __ballot(eq);
        const uint32_t c = sh.count[i * kEvictWaves + w];
        const int e = (int)(c >> 16) + __popcll(me & below), r = (int)(c & 0xFFFFu) + __popcll(mg & below) + min(e, need);
        if ((gt || (eq && e < need)) && r >= r_begin && r < r_end) sh.list[r - r_begin] = j;
      }
    } else {
      // waves take contiguous runs of slots
      const int run = ((old + kEvictWaves - 1) / kEvictWaves + 63) & ~63;
      const int a = min(w * run, old), b = min(a + run, old);
      int gt = 0, eq = 0;
#pragma unroll 4
      for (int j = a; j < b; j += 64) {
        const uint32_t k = j + lane < b ? order_key(mass[j + lane]) : 0u;
        gt += __popcll(__ballot(j + lane < b && k > prefix));
        eq += __popcll(__ballot(j + lane < b && k == prefix));
      }
      if (lane == 0) {
        sh.count[w] = gt;
        sh.count[kEvictWaves + w] = eq;
      }
      __syncthreads();
      gt = eq = 0;
      for (int x = 0; x < w; ++x) {
        gt += sh.count[x];
        eq += sh.count[kEvictWaves + x];
      }
#pragma unroll 4
      for (int j = a; j < b; j += 64) {
        const bool in = j + lane < b;
        const uint32_t k = in ? order_key(mass[j + lane]) : 0u;
        const uint64_t mg = __ballot(in && k > prefix), me = __ballot(in && k == prefix);
        const int e = eq + __popcll(me & below), r = gt + __popcll(mg & below) + min(e, need);
        const bool sel = in && (k > prefix || (k == prefix && e < need));
        if (sel && r >= r_begin && r < r_end) sh.list[r - r_begin] = j + lane;
        gt += __popcll(mg);
        eq += __popcll(me);
      }
    }
    __syncthreads();
  }
  auto source = [&](int r) { return !cut ? r : (r < from_old ? sh.list[r - r_begin] : old + (r - from_old)); };

  const int64_t head = (int64_t)s * p.KVH + kv;
  const int left_n = p.to_width << p.shift;
  for (int r = r_begin + tid; r < r_end; r += kEvictThreads) {
    const int j = r < kept_n ? source(r) : -1;
    p.kept[head * p.budget + r] = j;
    p.left[head * left_n + r] = j >= 0 ? mass[j] : 0.f;
  }
  if (part == parts - 1)
    for (int r = p.budget + tid; r < left_n; r += kEvictThreads) p.left[head * left_n + r] = 0.f;
  if (part == 0 && kv == 0 && tid == 0) p.new_lens[s] = kept_n;

  const int lanes = p.D / 8, mask = (1 << p.shift) - 1;   // 16-byte pieces of a slot
  const int32_t* row = p.table + (int64_t)s * p.ld_table;
  const int32_t* to = p.to + (int64_t)s * p.ld_to;
  const int piece = tid & (lanes - 1), step = kEvictThreads / lanes, end = min(r_end, kept_n);
#pragma unroll 4
  for (int r = r_begin + tid / lanes; r < end; r += step) {
    const int j = source(r), dst = to[r >> p.shift], page = paged_page(row, j, len, p.shift, p.pages);
    if (dst < 0 || dst >= p.pages) continue;
    u4 a = {}, b = {};   // a slot without a page moves as zeros
    if (page >= 0) {
      a = ((const u4*)((const uint16_t*)p.k.ptr + page * p.k.page + kv * p.k.head + (int64_t)(j & mask) * p.k.slot))[piece];
      b = ((const u4*)((const uint16_t*)p.v.ptr + page * p.v.page + kv * p.v.head + (int64_t)(j & mask) * p.v.slot))[piece];
    }
    ((u4*)((uint16_t*)const_cast<void*>(p.k.ptr) + dst * p.k.page + kv * p.k.head + (int64_t)(r & mask) * p.k.slot))[piece] = a;
    ((u4*)((uint16_t*)const_cast<void*>(p.v.ptr) + dst * p.v.page + kv * p.v.head + (int64_t)(r & mask) * p.v.slot))[piece] = b;
  }
}

}  // namespace

hipError_t prope_launch(const PagedRopeArgs& a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  const int chunks_log = a.D == 128 ? 3 : 2, heads = a.H + 2 * a.KVH;
  // threads per token and frequency chunk: enough of them to fill the chip
  const int64_t want = ((int64_t)1 << 18) / ((int64_t)a.rows << chunks_log);
  const int split = (int)std::max<int64_t>(1, std::min<int64_t>(heads, want));
  const int64_t grid = ((((int64_t)a.rows * split) << chunks_log) + 255) / 256;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  if (a.bf16) paged_rope_kernel<BF16><<<(int)grid, 256, 0, s>>>(a, split, chunks_log);
  else paged_rope_kernel<F16><<<(int)grid, 256, 0, s>>>(a, split, chunks_log);
  return hipGetLastError();
}

hipError_t pevict_launch(const PagedEvictArgs& a, int num_cus, hipStream_t s) {
  const int64_t rows = (int64_t)a.b * a.KVH;
  if (rows == 0) return hipSuccess;
  // parts of a head: lists that fit, and about a workgroup per CU of at least 64
  // slots each (two per CU, where the long heads' registers let one run at a
  // time: 159 against 143 us for eight sequences of 20-32k slots)
  int64_t parts = std::max<int64_t>((a.budget + kEvictList - 1) / kEvictList,
                                    std::min<int64_t>(num_cus / rows, (a.budget + 63) / 64));
  if (parts < 1) parts = 1;
  const int per = (int)((a.budget + parts - 1) / parts);
  if (rows * parts > 0x7fffffff) return hipErrorInvalidValue;
  const int grid = (int)(rows * parts);
  if (a.cap <= 4 * kEvictThreads) paged_evict_kernel<4><<<grid, kEvictThreads, 0, s>>>(a, (int)parts, per);
  else if (a.cap <= 32 * kEvictThreads) paged_evict_kernel<32><<<grid, kEvictThreads, 0, s>>>(a, (int)parts, per);
  else paged_evict_kernel<0><<<grid, kEvictThreads, 0, s>>>(a, (int)parts, per);
  return hipGetLastError();
}

}  // namespace mq
