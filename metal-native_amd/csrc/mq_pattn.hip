// Attention of new tokens over a paged key/value cache.
//
// Row r of a sequence's key/value head is query head r % g of its chunk's
// token r / g (g query heads share the key/value head).  For a row at position
// p and the slots j that it sees,
//   x_j = scale * q . k_j,  x_j <- cap * tanh(x_j / cap),  x_j <- x_j - slope * |p - j|
//   out = sum_j exp(x_j) v_j / sum_j exp(x_j),   lse = log sum_j exp(x_j)
// in one pass over the slots: with a reference M, the sums of exp2(x_j - M)
// v_j and exp2(x_j - M) (x in units of log 2) are multiplied by exp2(M - M')
// where M moves to M'.  M moves only when a score passes it by kAbove: then to
// kBelow under the row's largest score, so that weights reach from 2^15 down,
// far enough into fp16's range that 2^17 weights which round to zero together
// stay below an output's rounding step.  Weights are rounded to the cache's type for
// the product with v (the matrix instruction takes no other); their sum, the
// output's sum and M are fp32.
//
// Both products are v_mfma_f32_32x32x16 with keys (then value columns) as the
// result's rows and 32 query rows as its columns: S^T = K Q^T leaves lane l the
// scores of row l % 32 for the slots 8i + 4 (l / 32) + 0..3, which is the order
// in which O^T = V^T P^T may take its 16 slots per step, so weights go from one
// product to the next without leaving their lane, and a row's maximum and sum
// are one exchange between two lanes.  V^T comes from LDS by the transposing
// read (ds_read_b64_tr_b16).  Tiles of K and V reach LDS by buffer loads that
// bypass registers; a page's part of a tile has a descriptor of its own whose
// range ends at the sequence's last slot, so that what lies beyond, and what
// pages outside the cache would hold, arrives as zeros.
#include "mq_paged_dev.hpp"

#include <algorithm>

namespace mq {
namespace {

constexpr float kAbove = 15.f, kBelow = 7.f;

// What a wave knows of its 32 rows.
struct Rows {
  int pos;              // position of the lane's row; padding rows see nothing
  int first, last;      // positions of the wave's first and last row (uniform)
  float slope2;         // slope * log2(e) of the lane's head
};

template <int D> struct Acc {
  f16v o[D / 32];
  float m, l;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = (f16v){};
    m = -3.0e38f;
    l = 0.f;
  }
};

// Whether any of n 16-byte pieces in LDS holds an infinity or NaN (n a
// multiple of 64; wave-uniform): an exponent of ones carries into the sign's place.
template <typename T> __device__ __forceinline__ bool not_finite(const u4* at, int n) {
  uint32_t any = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < n; i += 64) {
    const u4 v = at[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= (v[e] & T::kExp) + T::kExpLow;
  }
  return __any((any & 0x80008000u) != 0);
}

// The values with zeros for infinities and NaN.
template <typename T> __device__ __forceinline__ u4 finite(u4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t bad = ((v[e] & T::kExp) + T::kExpLow) & 0x80008000u;   // the sign bits' places
    v[e] &= ~((bad >> 15) * 0xFFFFu);
  }
  return v;
}

// One tile of 32 * NB slots from tile0 for the wave's rows.  vm: bit per slot,
// set where it exists.
template <typename T, int D, int NB, bool EXTRA>
__device__ __forceinline__ void tile(const PagedArgs& p, const Rows& rw, const PagedSeq& sq, const u4 (&q)[D / 16],
                                     Acc<D>& ac, const u4* kt, const u4* vt, int tile0, uint64_t vm) {
  constexpr int ROW = Lay<D>::ROW;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  f16v s[NB];
  {
    const int swz = Lay<D>::swz_k(col) ^ h;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb] = (f16v){};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb] = T::mfma(kt[(32 * nb + col) * ROW + (swz ^ (2 * ks))], q[ks], s[nb]);
  }
  float c = p.scale * kLog2e;
  if constexpr (EXTRA) {
    const float cap = p.softcap;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float x = s[nb][j] * p.scale;
        if (cap != 0.f) {
          const float e = __builtin_amdgcn_exp2f(x * (2.f * kLog2e / cap));   // tanh y = 1 - 2 / (e^2y + 1)
          x = cap - 2.f * cap * __builtin_amdgcn_rcpf(e + 1.f);
        }
        const int away = rw.pos - (tile0 + 32 * nb + 8 * (j / 4) + 4 * h + j % 4);
        s[nb][j] = x * kLog2e - rw.slope2 * fabsf((float)away);
      }
    c = 1.f;
  }
  constexpr uint64_t kAll = NB == 2 ? ~0ull : 0xFFFFFFFFull;
  const int end = tile0 + 32 * NB - 1;
  const bool masked = vm != kAll || end > rw.first || (p.window > 0 && (int64_t)tile0 <= (int64_t)rw.last - p.window);
  if (masked) {
    const int64_t lo64 = p.window > 0 ? (int64_t)rw.pos - p.window + 1 : -0x7fffffff;
    const int hi = rw.pos - tile0 - 4 * h, lo = (int)(lo64 < -0x7fffffff ? -0x7fffffff : lo64), pre = sq.prefix - tile0 - 4 * h;
    const int lor = lo < 0 ? -0x7fffffff : lo - tile0 - 4 * h;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t bits = (uint32_t)(vm >> (32 * nb)) >> (4 * h);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int kk = 8 * (j / 4) + j % 4, jj = 32 * nb + kk;
        const bool see = ((jj <= hi && jj >= lor) || jj < pre) && ((bits >> kk) & 1);
        s[nb][j] = see ? s[nb][j] : -INFINITY;
      }
    }
  }
  float t = s[0][0];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < 16; ++j) t = fmaxf(t, s[nb][j]);
  t = fmaxf(t, swap32(t)) * c;
  if (__any(t > ac.m + kAbove)) {
    const float m2 = t > ac.m + kAbove ? t - kBelow : ac.m;
    const float f = __builtin_amdgcn_exp2f(ac.m - m2);
    ac.m = m2;
    ac.l *= f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) ac.o[i] *= f;
  }
  const float nm = -ac.m;
  float l = 0.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[nb][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][j], c, nm));
      l += s[nb][j];
    }
  ac.l += l;
  const int i = lane & 15, key0 = 4 * h + (i >> 2), low = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  const s4* vp = (const s4*)vt + key0 * (D / 4) + (i & 1);
  const int sv = Lay<D>::swz_v(key0);
  auto weights = [&](int u) {
    u4 pr;
#pragma unroll
    for (int e = 0; e < 4; ++e) pr[e] = pack2<T>(s[u / 2][8 * (u & 1) + 2 * e], s[u / 2][8 * (u & 1) + 2 * e + 1]);
    return pr;
  };
  auto values = [&](int u, int db) {
    const s4* a = vp + 16 * u * (D / 4) + 2 * ((4 * db + low) ^ sv);
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)a);
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(a + 8 * (D / 4)));
    return __builtin_bit_cast(u4, (s8v)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  if (masked && not_finite<T>(vt, 32 * NB * Lay<D>::ROW)) {
    // A hidden slot's infinity or NaN times its weight of zero would be NaN:
    // the product takes zeros for them all, and each is then added to the
    // rows that see its slot (times any weight it is itself, or NaN).
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u) {
      const u4 pr = weights(u);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) ac.o[db] = T::mfma(finite<T>(values(u, db)), pr, ac.o[db]);
    }
#pragma unroll 1
    for (int kk = 0; kk < 32 * NB; ++kk) {
      const bool see = paged_visible(rw.pos, tile0 + kk, sq.len, sq.prefix, p.window) && ((vm >> kk) & 1);
      const uint2* row = (const uint2*)(vt + kk * Lay<D>::ROW);
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint2 raw = row[2 * ((4 * db + e) ^ Lay<D>::swz_v(kk)) + h];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t bits = (x < 2 ? raw.x : raw.y) >> (16 * (x & 1)) & 0xFFFFu;
            if (see && (bits & (T::kExp & 0xFFFFu)) == (T::kExp & 0xFFFFu))
              ac.o[db][4 * e + x] += (float)__builtin_bit_cast(typename T::e, (uint16_t)bits);
          }
        }
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < 2 * NB; ++u) {
    const u4 pr = weights(u);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) ac.o[db] = T::mfma(values(u, db), pr, ac.o[db]);
  }
}

// The wave's rows r0 .. r0 + 32 of a sequence and key/value head, and their
// queries (zeros for padding rows).
template <int D>
__device__ __forceinline__ Rows load_rows(const PagedArgs& p, const PagedSeq& sq, int kv, int r0, u4 (&q)[D / 16]) {
  const int lane = threadIdx.x & 63, r = r0 + (lane & 31), h = lane >> 5;
  const int i = (int)p.gdiv.div((uint32_t)r), a = kv * p.g + r - i * p.g, total = sq.n * p.g;
  const bool have = r < total;
  Rows rw;
  rw.pos = sq.len - sq.n + i;
  rw.first = uni(rw.pos);
  const int rl = (r0 + 31 < total ? r0 + 31 : total - 1);
  rw.last = sq.len - sq.n + (int)p.gdiv.div((uint32_t)(rl < 0 ? 0 : rl));
  rw.slope2 = p.slopes && have ? p.slopes[a] * kLog2e : 0.f;
  const u4* src = (const u4*)((const uint16_t*)p.q + (int64_t)(sq.start + i) * p.q_t + (int64_t)a * p.q_h) + h;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) q[ks] = have ? src[2 * ks] : (u4){0u, 0u, 0u, 0u};
  // waited for here: the compiler would otherwise wait in the loop over the
  // tiles, where the wait takes in the loads of the next tile
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" : "+v"(q[ks]));
  return rw;
}

template <typename T>
__device__ __forceinline__ void store4(void* out, int64_t at, f4 v) {
  const uint64_t w = pack2<T>(v[0], v[1]) | (uint64_t)pack2<T>(v[2], v[3]) << 32;
  *(uint64_t*)((uint16_t*)out + at) = w;
}
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float m, float l) {
  return l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- many rows: one workgroup per 128 rows, whose four waves share the tiles ----

constexpr int kRowsP = 128;

template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(PagedArgs p) {
  constexpr int TK = 64, ROW = Lay<D>::ROW, GS = Lay<D>::GS, NG = TK / GS / 4;
  __shared__ u4 k0[TK * ROW], k1[TK * ROW], v0[TK * ROW], v1[TK * ROW];
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6);
  const int kv = blockIdx.x % p.KVH;
  int item = blockIdx.x / p.KVH, seq = -1;
  PagedSeq sq{};
  for (int s0 = 0; s0 < p.b && seq < 0; s0 += 64) {
    const int s = s0 + lane;
    PagedSeq mine{};
    if (s < p.b) mine = load_seq(p, s);
    const int tiles = (int)(((int64_t)mine.n * p.g + kRowsP - 1) / kRowsP);
    const int64_t sum = wave_scan(tiles);
    const uint64_t past = __ballot(sum > item);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      seq = s0 + at;
      sq.start = __builtin_amdgcn_readlane(mine.start, at);
      sq.n = __builtin_amdgcn_readlane(mine.n, at);
      sq.len = __builtin_amdgcn_readlane(mine.len, at);
      sq.prefix = __builtin_amdgcn_readlane(mine.prefix, at);
      // last rows first: they see most
      item = (int)__builtin_amdgcn_readlane((int)sum, at) - 1 - item;
    } else {
      item -= __builtin_amdgcn_readlane((int)sum, 63);
    }
  }
  if (seq < 0) return;

  const int r0 = item * kRowsP, total = sq.n * p.g, off = sq.len - sq.n;
  u4 q[D / 16];
  const Rows rw = load_rows<D>(p, sq, kv, r0 + 32 * w, q);
  const bool busy = r0 + 32 * w < total;
  const int rl = r0 + kRowsP < total ? r0 + kRowsP - 1 : total - 1;
  const PagedSpan span = paged_span(off + (int)p.gdiv.div(r0), off + (int)p.gdiv.div(rl), sq.len, sq.prefix, p.window, TK);
  const int count = span.count();

  const Base kb = cache_base(p.k, kv), vb = cache_base(p.v, kv);
  const int gl = lane / ROW, piece = lane % ROW;
  const uint32_t koff = gl * kb.slot + 16u * (piece ^ Lay<D>::swz_k(GS * w + gl));
  const uint32_t voff = gl * vb.slot + 16u * (piece ^ Lay<D>::swz_v(GS * w + gl));
  const int32_t* row = p.table + (int64_t)seq * p.ld_table;
  const int mask = (1 << p.shift) - 1;
  // the table's entry for the lane's slot in tile i, checked when it is used:
  // a check here would wait for the loads before it
  auto entry_of = [&](int i) {
    const int j = span.tile(i < count ? i : count - 1) * TK + lane;
    return row[(j < sq.len ? j : sq.len - 1) >> p.shift];
  };
  auto page_of = [&](int i, int id) {
    return i < count && span.tile(i) * TK + lane < sq.len && id >= 0 && id < p.pages ? id : -1;
  };
  auto load = [&](int i, int pg, uint64_t vm, u4* kd, u4* vd) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int gi = 4 * n + w, j = gi * GS;
      const int page = __builtin_amdgcn_readlane(pg, j), nv = __popcll((vm >> j) & ((1u << GS) - 1));
      const int in = (span.tile(i) * TK + j) & mask;
      load_group(kb, page, in, nv, koff, kd + 64 * gi);
      load_group(vb, page, in, nv, voff, vd + 64 * gi);
    }
  };

  Acc<D> ac;
  ac.clear();
  int id = 0;
  uint64_t vm = 0;
  if (count > 0) {
    const int pg = page_of(0, entry_of(0));
    vm = __ballot(pg >= 0);
    load(0, pg, vm, k0, v0);
    id = entry_of(1);
  }
  auto step = [&](int i, const u4* kt, const u4* vt, u4* kn, u4* vn) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();   // tile i is in LDS, and no wave reads tile i - 1 any more
    asm volatile("" ::: "memory");
    const int pg = page_of(i + 1, id);
    const uint64_t vm1 = __ballot(pg >= 0);
    if (i + 1 < count) {
      load(i + 1, pg, vm1, kn, vn);
      id = entry_of(i + 2);
    }
    const int t0 = span.tile(i) * TK;
    if (busy && (t0 <= rw.last || t0 < sq.prefix)) tile<T, D, 2, EXTRA>(p, rw, sq, q, ac, kt, vt, t0, vm);
    vm = vm1;
  };
  for (int i = 0; i < count; i += 2) {
    step(i, k0, v0, k1, v1);
    if (i + 1 < count) step(i + 1, k1, v1, k0, v0);
  }
  if (!busy) return;
  const int r = r0 + 32 * w + (lane & 31), h = lane >> 5;
  if (r >= total) return;
  const float l = ac.l + swap32(ac.l), f = inverse(l);
  const int tok = (int)p.gdiv.div(r), a = kv * p.g + r - tok * p.g;
  const int64_t at = (int64_t)(sq.start + tok) * p.H + a;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16v& o = ac.o[db];
      store4<T>(p.out, at * D + 32 * db + 8 * e + 4 * h,
                (f4){o[4 * e] * f, o[4 * e + 1] * f, o[4 * e + 2] * f, o[4 * e + 3] * f});
    }
  if (p.lse && h == 0) p.lse[at] = log_sum(ac.m, l);
}

// ---- few rows: every workgroup takes an equal run of (row block, key tile)
// units, its four waves the run's tiles in turn ----

constexpr int kRowsS = 32, kTileS = 32;

__device__ __forceinline__ int64_t split_units(const PagedArgs& p, const PagedSeq& q, int* blocks, PagedSpan* span) {
  *blocks = (int)(((int64_t)q.n * p.g + kRowsS - 1) / kRowsS);
  *span = paged_span(q.len - q.n, q.len - 1, q.len, q.prefix, p.window, kTileS);
  const int c = span->count();
  return (int64_t)*blocks * (c > 0 ? c : 1);   // a row that sees nothing is written too
}
__device__ __forceinline__ int64_t all_units(const PagedArgs& p) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int s0 = 0; s0 < p.b; s0 += 64) {
    int blocks;
    PagedSpan span;
    const int64_t u = s0 + lane < p.b ? split_units(p, load_seq(p, s0 + lane), &blocks, &span) : 0;
    total += uni64(__shfl(wave_scan(u), 63));
  }
  return total;
}
// units per workgroup: at least one tile per wave
__device__ __forceinline__ int64_t units_per(int64_t units, int kvh, int wgs) {
  const int64_t per = (units * kvh + wgs - 1) / wgs;
  return per < 4 ? 4 : per;
}
constexpr int record_floats(int D) { return kRowsS * (D + 2); }

template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(256, 1) void paged_split_kernel(PagedArgs p, float* ws, int wgs) {
  constexpr int TK = kTileS, ROW = Lay<D>::ROW, GS = Lay<D>::GS, NG = TK / GS;
  __shared__ u4 k0[4 * TK * ROW], k1[4 * TK * ROW], v0[4 * TK * ROW], v1[4 * TK * ROW];
  __shared__ float ml[4][kRowsS][2];
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
  const int64_t units = all_units(p), per = units_per(units, p.KVH, wgs);
  const int64_t u_begin = per * blockIdx.x, u_all = units * p.KVH;
  const int64_t u_end = u_begin + per < u_all ? u_begin + per : u_all;
  const int gl = lane / ROW, piece = lane % ROW;
  const int mask = (1 << p.shift) - 1;
  u4* const kw[2] = {k0 + w * TK * ROW, k1 + w * TK * ROW};
  u4* const vw[2] = {v0 + w * TK * ROW, v1 + w * TK * ROW};

  for (int64_t u = u_begin; u < u_end;) {
    const int kv = uni((int)(u / units));
    int64_t left = u - kv * units;
    int seq = -1, blocks = 0;
    PagedSeq sq{};
    PagedSpan span{};
    for (int s0 = 0; s0 < p.b && seq < 0; s0 += 64) {
      PagedSeq mine{};
      int64_t n = 0;
      if (s0 + lane < p.b) {
        mine = load_seq(p, s0 + lane);
        n = split_units(p, mine, &blocks, &span);
      }
      const int64_t sum = wave_scan(n);
      const uint64_t past = __ballot(sum > left);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        left -= uni64(__shfl(sum - n, at));
        seq = s0 + at;
        sq.start = __builtin_amdgcn_readlane(mine.start, at);
        sq.n = __builtin_amdgcn_readlane(mine.n, at);
        sq.len = __builtin_amdgcn_readlane(mine.len, at);
        sq.prefix = __builtin_amdgcn_readlane(mine.prefix, at);
      } else {
        left -= uni64(__shfl(sum, 63));
      }
    }
    if (seq < 0) return;   // not reached: u < u_all
    split_units(p, sq, &blocks, &span);
    const int count = span.count(), cost = count > 0 ? count : 1;
    const int block = uni((int)(left / cost)), t_begin = uni((int)(left - (int64_t)block * cost));
    const int t_end = uni((int)(cost - t_begin < u_end - u ? cost : t_begin + (u_end - u)));
    const bool whole = t_begin == 0 && t_end == cost;

    u4 q[D / 16];
    const int r0 = block * kRowsS, total = sq.n * p.g;
    const Rows rw = load_rows<D>(p, sq, kv, r0, q);
    const Base kb = cache_base(p.k, kv), vb = cache_base(p.v, kv);
    const int32_t* row = p.table + (int64_t)seq * p.ld_table;
    const int last = t_end < count ? t_end : count;
    auto entry_of = [&](int i) {
      const int j = span.tile(i < last ? i : last - 1) * TK + (lane & 31);
      return row[(j < sq.len ? j : sq.len - 1) >> p.shift];
    };
    auto page_of = [&](int i, int id) {
      return i < last && lane < TK && span.tile(i) * TK + lane < sq.len && id >= 0 && id < p.pages ? id : -1;
    };
    auto load = [&](int i, int pg, uint64_t vm, u4* kd, u4* vd) {
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        const int j = gi * GS;
        const int page = __builtin_amdgcn_readlane(pg, j), nv = __popcll((vm >> j) & ((1u << GS) - 1));
        const int in = (span.tile(i) * TK + j) & mask;
        load_group(kb, page, in, nv, gl * kb.slot + 16u * (piece ^ Lay<D>::swz_k(j + gl)), kd + 64 * gi);
        load_group(vb, page, in, nv, gl * vb.slot + 16u * (piece ^ Lay<D>::swz_v(j + gl)), vd + 64 * gi);
      }
    };
    Acc<D> ac;
    ac.clear();
    int i = t_begin + w;
    int id = 0;
    uint64_t vm = 0;
    if (i < last) {
      const int pg = page_of(i, entry_of(i));
      vm = __ballot(pg >= 0);
      load(i, pg, vm, kw[0], vw[0]);
      id = entry_of(i + 4);
    }
    auto step = [&](int n, const u4* kt, const u4* vt, u4* kn, u4* vn) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // the wave's own tile is in LDS
      const int pg = page_of(n + 4, id);
      const uint64_t vm1 = __ballot(pg >= 0);
      if (n + 4 < last) {
        load(n + 4, pg, vm1, kn, vn);
        id = entry_of(n + 8);
      }
      tile<T, D, 1, EXTRA>(p, rw, sq, q, ac, kt, vt, span.tile(n) * TK, vm);
      vm = vm1;
    };
    for (; i < last; i += 8) {
      step(i, kw[0], vw[0], kw[1], vw[1]);
      if (i + 4 < last) step(i + 4, kw[1], vw[1], kw[0], vw[0]);
    }

    // ---- the four waves' sums meet in LDS: f4 piece d / 4 of row r at [d / 4][r] ----
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    {
      const int r = lane & 31, h = lane >> 5;
      const float l = ac.l + swap32(ac.l);
      if (h == 0) {
        ml[w][r][0] = ac.m;
        ml[w][r][1] = l;
      }
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f4* at = (f4*)(db < D / 64 ? kw[0] : kw[1]) + ((db % (D / 64)) * 8 + 2 * e + h) * kRowsS + r;
          *at = (f4){ac.o[db][4 * e], ac.o[db][4 * e + 1], ac.o[db][4 * e + 2], ac.o[db][4 * e + 3]};
        }
    }
    __syncthreads();
    {
      const int r = tid & 31;
      float m = ml[0][r][0];
#pragma unroll
      for (int x = 1; x < 4; ++x) m = fmaxf(m, ml[x][r][0]);
      float f[4], l = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        f[x] = __builtin_amdgcn_exp2f(ml[x][r][0] - m);
        l += ml[x][r][1] * f[x];
      }
      const float inv = inverse(l);
      float* rec = ws + ((int64_t)2 * blockIdx.x + (u == u_begin ? 0 : 1)) * record_floats(D);
      const int tok = (int)p.gdiv.div(r0 + r), a = kv * p.g + r0 + r - tok * p.g;
      const int64_t at = (int64_t)(sq.start + tok) * p.H + a;
      const bool have = r0 + r < total;
#pragma unroll
      for (int n = 0; n < D / 32; ++n) {
        const int d4 = (tid >> 5) + 8 * n;
        f4 v = {};
        if (have) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            v += f[x] * ((const f4*)((n < D / 64 ? k0 : k1) + x * TK * ROW))[(d4 % (D / 8)) * kRowsS + r];
          if (whole) store4<T>(p.out, at * D + 4 * d4, v * inv);
          else *(f4*)(rec + 4 * (d4 * kRowsS + r)) = v;
        }
      }
      if (have && tid < kRowsS) {
        if (!whole) {
          rec[kRowsS * D + 2 * r] = m;
          rec[kRowsS * D + 2 * r + 1] = l;
        } else if (p.lse) {
          p.lse[at] = log_sum(m, l);
        }
      }
    }
    __syncthreads();
    u += t_end - t_begin;
  }
}

// Adds up the records of the row blocks that more than one workgroup worked
// on, in the workgroups' order.  blockIdx.x: row block and key/value head;
// blockIdx.y: 32 of the output's columns.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs p, const float* ws, int wgs) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t units = all_units(p), per = units_per(units, p.KVH, wgs);
  const int kv = blockIdx.x % p.KVH;
  int item = blockIdx.x / p.KVH, seq = -1, blocks = 0;
  int64_t u0 = kv * units;
  PagedSeq sq{};
  PagedSpan span{};
  for (int s0 = 0; s0 < p.b && seq < 0; s0 += 64) {
    PagedSeq mine{};
    int64_t n = 0;
    int nb = 0;
    if (s0 + lane < p.b) {
      mine = load_seq(p, s0 + lane);
      n = split_units(p, mine, &nb, &span);
    }
    const int64_t sum = wave_scan(nb), usum = wave_scan(n);
    const uint64_t past = __ballot(sum > item);
    const int at = past ? __ffsll((unsigned long long)past) - 1 : 63;
    if (past) {
      item -= uni((int)__shfl(sum - nb, at));
      u0 += uni64(__shfl(usum - n, at));
      seq = s0 + at;
      sq.start = __builtin_amdgcn_readlane(mine.start, at);
      sq.n = __builtin_amdgcn_readlane(mine.n, at);
      sq.len = __builtin_amdgcn_readlane(mine.len, at);
      sq.prefix = __builtin_amdgcn_readlane(mine.prefix, at);
    } else {
      item -= uni((int)__shfl(sum, 63));
      u0 += uni64(__shfl(usum, 63));
    }
  }
  if (seq < 0) return;
  split_units(p, sq, &blocks, &span);
  const int cost = span.count() > 0 ? span.count() : 1;
  u0 += (int64_t)item * cost;
  const int64_t u1 = u0 + cost;
  const int64_t w0 = u0 / per, w1 = (u1 - 1) / per;
  if (w0 == w1) return;
  const int r = tid & 31, r0 = item * kRowsS, d4 = blockIdx.y * 8 + (tid >> 5);
  if (r0 + r >= sq.n * p.g) return;
  auto record = [&](int64_t w) {   // the workgroup's first segment, but where the block starts inside its run
    return ws + (2 * w + (w == w0 && w * per != u0 ? 1 : 0)) * record_floats(D);
  };
  float m = -3.0e38f;
  for (int64_t w = w0; w <= w1; ++w) m = fmaxf(m, record(w)[kRowsS * D + 2 * r]);
  f4 v = {};
  float l = 0.f;
#pragma unroll 4
  for (int64_t w = w0; w <= w1; ++w) {
    const float* rec = record(w);
    const float f = __builtin_amdgcn_exp2f(rec[kRowsS * D + 2 * r] - m);
    l += rec[kRowsS * D + 2 * r + 1] * f;
    v += f * *(const f4*)(rec + 4 * (d4 * kRowsS + r));
  }
  const int tok = (int)p.gdiv.div(r0 + r), a = kv * p.g + r0 + r - tok * p.g;
  const int64_t at = (int64_t)(sq.start + tok) * p.H + a;
  store4<T>(p.out, at * D + 4 * d4, v * inverse(l));
  if (p.lse && d4 == 0) p.lse[at] = log_sum(m, l);
}

int64_t row_blocks(const PagedArgs& a, int rows) {   // at most, over all sequences
  return ((int64_t)a.rows * a.g + rows - 1) / rows + (a.cu ? a.b : (int64_t)a.rows * ((a.g + rows - 1) / rows));
}
bool many_rows(const PagedArgs& a, int num_cus) {
  return ((int64_t)a.rows * a.g / kRowsP) * a.KVH >= num_cus;
}

template <typename T, int D>
hipError_t launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) {
  if (many_rows(a, num_cus)) {
    const int64_t grid = row_blocks(a, kRowsP) * a.KVH;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    if (a.extra()) paged_rows_kernel<T, D, true><<<(int)grid, 256, 0, s>>>(a);
    else paged_rows_kernel<T, D, false><<<(int)grid, 256, 0, s>>>(a);
    return hipGetLastError();
  }
  if (a.extra()) paged_split_kernel<T, D, true><<<num_cus, 256, 0, s>>>(a, (float*)ws, num_cus);
  else paged_split_kernel<T, D, false><<<num_cus, 256, 0, s>>>(a, (float*)ws, num_cus);
  const int64_t grid = row_blocks(a, kRowsS) * a.KVH;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  paged_join_kernel<T, D><<<dim3((int)grid, D / 32), 256, 0, s>>>(a, (const float*)ws, num_cus);
  return hipGetLastError();
}

}  // namespace

size_t pattn_workspace(const PagedArgs& a, int num_cus) {
  return many_rows(a, num_cus) ? 0 : (size_t)2 * num_cus * record_floats(a.D) * sizeof(float);
}

hipError_t pattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) {
  if (a.D == 128) return a.bf16 ? launch<BF16, 128>(a, num_cus, ws, s) : launch<F16, 128>(a, num_cus, ws, s);
  return a.bf16 ? launch<BF16, 64>(a, num_cus, ws, s) : launch<F16, 64>(a, num_cus, ws, s);
}

}  // namespace mq
