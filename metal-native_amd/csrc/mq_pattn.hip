// Attention of new tokens over a paged key/value cache.
//
// Row r of a sequence's key/value head is query head r % g of its chunk's
// token r / g (g query heads share the key/value head).  For a row at position
// p and the slots j that it sees,
//   x_j = scale * q . k_j,  x_j <- cap * tanh(x_j / cap),  x_j <- x_j - slope * |p - j|
//   out = sum_j exp(x_j) v_j / sum_j exp(x_j),   lse = log sum_j exp(x_j)
// in one pass over the slots: with a reference M, the sums of exp2(x_j - M)
// v_j and exp2(x_j - M) (x in units of log 2) are multiplied by exp2(M - M')
// where M moves to M'.  M moves only where weights would grow past 2^15 (few
// rows: a score more than kAbove over it; many rows: a lane's weights of a tile
// that add up to more): then to kBelow under the row's largest score, so that
// weights reach from 2^15 down, far enough into fp16's range that 2^17 weights
// which round to zero together stay below an output's rounding step.  Weights
// are rounded to the cache's type for the product with v (the matrix instruction
// takes no other); their sum, the output's sum and M are fp32.
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
  int pos;              // position of the lane's row (a padding row's queries are zeros, its results go nowhere)
  int first, last;      // positions of the wave's first and last row (uniform)
  float slope2;         // slope * log2(e) of the lane's head
};

template <int D> struct Acc {
  f16v o[D / 32];
  float m, l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = (f16v){};
    m = -3.0e38f;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ float sum() const {   // of both lanes of a row
    const float t = l[0] + l[1];
    return t + swap32(t);
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

// Cap and distance bias, in units of log 2: scores of 32 * NB slots from tile0.
template <int NB>
__device__ __forceinline__ void cap_and_bias(const PagedArgs& p, const Rows& rw, f16v (&s)[NB], int tile0) {
  const int h = (threadIdx.x & 63) >> 5;
  float scale = p.scale;
  if (p.softcap != 0.f) {
    cap_scores<true>(s, p);
    scale = 1.f;
  }
  scale *= kLog2e;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int away = rw.pos - (tile0 + 32 * nb + 8 * (j / 4) + 4 * h + j % 4);
      s[nb][j] = s[nb][j] * scale - rw.slope2 * fabsf((float)away);
    }
}

// Bits 0 .. n - 1, n clamped to 0 .. 64.
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0 : (n >= 64 ? ~0ull : (1ull << n) - 1); }

// -inf for what the lane's row does not see.  vm: bit per slot, set where it
// exists.  By a bit per slot, spread over the word, rather than by a condition
// per slot: those would all be kept in scalar registers at once.
template <int NB>
__device__ __forceinline__ void hide(const PagedArgs& p, const Rows& rw, const PagedSeq& sq, f16v (&s)[NB], int tile0, uint64_t vm) {
  const int h = (threadIdx.x & 63) >> 5;
  const int64_t before = p.window > 0 ? (int64_t)rw.pos - p.window + 1 - tile0 : 0;   // slots of the tile past the window
  uint64_t vis = low_bits(rw.pos - tile0 + 1) & ~low_bits(before > 64 ? 64 : (int)max(before, (int64_t)0));
  vis = ((vis | low_bits(sq.prefix - tile0)) & vm) >> (4 * h);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const uint32_t bits = (uint32_t)(vis >> (32 * nb));
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t see = (uint32_t)((int32_t)(bits << (31 - (8 * (j / 4) + j % 4))) >> 31);
      s[nb][j] = __uint_as_float((__float_as_uint(s[nb][j]) & see) | (0xFF800000u & ~see));
    }
  }
}

// Infinities and NaN among the values, of a tile that some row does not see
// all of: a hidden slot's would still be NaN times its weight of zero, so the
// products take zeros for them all, and the outputs that they reach are kept
// as bits (of the lane's D / 2 outputs of one row) and written at the end: up
// where a slot that the row sees holds +inf or NaN, down where -inf or NaN.
template <int D> struct Odd {
  uint64_t up, down;
  __device__ __forceinline__ void clear() { up = down = 0; }
  template <typename T>
  __device__ __forceinline__ void mark(const PagedArgs& p, const Rows& rw, const PagedSeq& sq, const u4* vt, int slots, int tile0,
                                       uint64_t vm) {
    const int h = (threadIdx.x & 63) >> 5;
    constexpr uint32_t kExp = T::kExp & 0xFFFFu;
#pragma unroll 1
    for (int kk = 0; kk < slots; ++kk) {
      const bool see = paged_visible(rw.pos, tile0 + kk, sq.len, sq.prefix, p.window) && ((vm >> kk) & 1);
      const uint16_t* row = (const uint16_t*)(vt + kk * Lay<D>::ROW);
#pragma unroll 1
      for (int i = 0; i < D / 2; ++i) {   // output i of the lane is 32 (i / 16) + 8 (i / 4 % 4) + 4 h + i % 4
        const uint32_t bits = row[8 * ((i >> 2) ^ Lay<D>::swz_v(kk)) + 4 * h + (i & 3)];
        const bool hit = see && (bits & kExp) == kExp, nan = (bits & 0x7FFFu) != kExp;
        up |= (uint64_t)(hit && (nan || !(bits & 0x8000u))) << i;
        down |= (uint64_t)(hit && (nan || (bits & 0x8000u))) << i;
      }
    }
  }
  __device__ __forceinline__ float fix(float v, int i) const {   // output i of the lane
    const bool a = (up >> i) & 1, b = (down >> i) & 1;
    return a ? (b ? __builtin_nanf("") : v + INFINITY) : (b ? v - INFINITY : v);
  }
};

// One tile of 32 * NB slots from tile0 for the wave's rows.  vm: bit per slot,
// set where it exists.  MASKED: some row may not see some slot of it.
//
// One wave's instructions issue in order, so both products read their LDS
// operands a few instructions ahead (kf, vf).
// keys_done() follows the last read of the keys, values_ready() comes before the
// first read of the values.
template <typename T, int D, int NB, bool EXTRA, bool MASKED, typename F, typename G>
__device__ __forceinline__ void tile(const PagedArgs& p, const Rows& rw, const PagedSeq& sq, const u4 (&q)[D / 16],
                                     Acc<D>& ac, Odd<D>& odd, const u4* kt, const u4* vt, int tile0, uint64_t vm,
                                     F&& keys_done, G&& values_ready) {
  constexpr int ROW = Lay<D>::ROW, KS = D / 16, DB = D / 32;
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  f16v s[NB];
  {
    const int swz = Lay<D>::swz_k(col) ^ h;
    const u4* kp = kt + col * ROW;
    constexpr int AHEAD = 3;   // steps of keys in flight
    u4 kf[AHEAD][NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb] = (f16v){};
#pragma unroll
    for (int ks = 0; ks < AHEAD; ++ks)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) kf[ks][nb] = kp[32 * nb * ROW + (swz ^ (2 * ks))];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb] = T::mfma(kf[ks % AHEAD][nb], q[ks], s[nb]);
      if (ks + AHEAD < KS) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) kf[ks % AHEAD][nb] = kp[32 * nb * ROW + (swz ^ (2 * (ks + AHEAD)))];
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * NB, 0);   // LDS reads
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);         // MFMAs
      if (ks + AHEAD < KS) __builtin_amdgcn_sched_group_barrier(0x100, NB, 0);
    }
  }
  const int i = lane & 15, key0 = 4 * h + (i >> 2), low = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
  const s4* vp = (const s4*)vt + key0 * (D / 4) + (i & 1);
  const int sv = Lay<D>::swz_v(key0);
  auto values = [&](int u, int db) {
    const s4* a = vp + 16 * u * (D / 4) + 2 * ((4 * db + low) ^ sv);
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)a);
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(a + 8 * (D / 4)));
    return __builtin_bit_cast(u4, (s8v)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  keys_done();
  values_ready();
  constexpr int VF = DB;   // the first step's values: on their way during the softmax
  u4 vf[VF];
#pragma unroll
  for (int x = 0; x < VF; ++x) vf[x] = values(x / DB, x % DB);
  asm volatile("" ::: "memory");   // not moved down to their use

  float c = p.scale * kLog2e;
  if constexpr (EXTRA) {
    cap_and_bias(p, rw, s, tile0);
    c = 1.f;
  }
  if constexpr (MASKED) hide(p, rw, sq, s, tile0, vm);
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
    ac.l[0] *= f;
    ac.l[1] *= f;
#pragma unroll
    for (int i = 0; i < DB; ++i) ac.o[i] *= f;
  }
  const float nm = -ac.m;
  float(&l)[2] = ac.l;
  auto weights = [&](int u) {
    u4 pr;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + 2 * e], c, nm));
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + 2 * e + 1], c, nm));
      l[0] += x;
      l[1] += y;
      pr[e] = pack2<T>(x, y);
    }
    return pr;
  };
  if (MASKED && not_finite<T>(vt, 32 * NB * ROW)) {
    odd.template mark<T>(p, rw, sq, vt, 32 * NB, tile0, vm);
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u) {
      const u4 pr = weights(u);
#pragma unroll
      for (int db = 0; db < DB; ++db) ac.o[db] = T::mfma(finite<T>(values(u, db)), pr, ac.o[db]);
    }
    return;
  }
  u4 pr = weights(0);
#pragma unroll
  for (int u = 0; u < 2 * NB; ++u) {
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      ac.o[db] = T::mfma(vf[db], pr, ac.o[db]);
      if (u + 1 < 2 * NB) vf[db] = values(u + 1, db);
    }
    if (u + 1 < 2 * NB) pr = weights(u + 1);
  }
#pragma unroll
  for (int u = 0; u < 2 * NB; ++u)
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (u + 1 < 2 * NB) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 28 / DB, 0);
      }
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
  return rw;
}
// Waits for them: the compiler would otherwise wait in the loop over the tiles,
// where the wait takes in the loads of the next tile.
template <int N> __device__ __forceinline__ void have_queries(u4 (&q)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(q[i]));
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

// Tokens of no chunk (before the first one, past the last) give what a row that
// sees nothing gives.  A call with chunk offsets launches for more blocks of ROWS
// rows than there can be: b more than all its rows fill, of which b chunks waste
// less than b.  So the workgroups that find no block are enough to take ROWS rows
// of these tokens each, this one the at-th.
template <int D, int ROWS>
__device__ __forceinline__ void clear_unused(int kv, int at) {
  // the arguments (a kernel's first) once more from where they lie: kept in
  // registers for this they cost the 64-wide few-row kernel one of its three
  // waves (five masked chunks 42.0 us, 47.2 so)
  uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const PagedArgs& p = *(const PagedArgs*)args;
  if (!p.cu) return;
  const int lo = min(max(p.cu[0], 0), p.rows), skip = min(max(p.cu[p.b], lo), p.rows) - lo;
  const int per = (ROWS + p.g - 1) / p.g;
#pragma unroll 1
  for (int o = at * per; o < (at + 1) * per && o < p.rows - skip; ++o) {
    const int64_t head = (int64_t)(o < lo ? o : o + skip) * p.H + kv * p.g;
#pragma unroll 1
    for (int c = threadIdx.x; c < p.g * (D / 8); c += blockDim.x) {   // 16 bytes each
      *(u4*)((uint16_t*)p.out + head * D + 8 * c) = (u4){0u, 0u, 0u, 0u};
      if (p.lse && c < p.g) p.lse[head + c] = -INFINITY;
    }
  }
}

// ---- many rows: one workgroup of eight waves per 256 rows ----
//
// Per tile of 64 slots a wave has D / 4 MFMAs (output of the tile before,
// scores of this one) and a softmax of about as many cycles.  One wave issues
// an instruction every five cycles at most, so one per SIMD cannot keep both
// units busy; two can, if one multiplies while the other takes the softmax.
// Waves 0..3 and 4..7 (one of each per SIMD) therefore stand half a tile apart
// and change places at a barrier: phase 2t is waves 0..3's products of tile t,
// phase 2t + 1 their softmax, and waves 4..7 are one phase behind.
//
// Tiles of keys lie in four LDS slots, of values (read a tile later) in five.  A
// wave asks for its eight slots of tile t + 3 among its products of tile t, whose
// issue slots are free (beside the softmax the loads' address arithmetic took 230
// of 1900 cycles), and waits for them before its products of tile t + 2.
//
// 4096 tokens of 28 heads over 4, 128 wide, fp16, behind 28672 slots: 1.63-1.72 ms,
// 1.05-1.11 PFLOP/s where a large matrix product reaches 1.35.  On the way: four
// waves of 32 rows with two tiles in flight 2.30 ms; eight in two groups 1.79;
// no maximum beforehand 1.69; three tiles ahead 1.63.  What bounds it then is the
// count of workgroups: 448 on 256 CUs, one each, are two rounds of which the
// second is three quarters full (rows_plan says why they are not split).  Seven prompts of 300 to 2048 tokens: 79 us for
// 48 GFLOP, of which the longest workgroup's 32 tiles take 55.

constexpr int kRowsP = 256, kTileP = 64, kPerMinP = 8;   // kPerMinP: fewest tiles of a part

// Tiles per part of a row block that sees `count`: parts_max parts, but of
// per_min tiles at least.
__device__ __forceinline__ int tiles_per_part(int count, int parts_max, int per_min) {
  const int per = ((count + parts_max - 1) / parts_max + 3) & ~3;
  return uni(per < per_min ? per_min : per);
}

// Partial sums of a part: R rows (the call's most rows per block, a multiple of
// eight) of D outputs, then R (m, l) pairs.
__device__ __host__ constexpr int record_floats(int D, int R) { return R * (D + 2); }

template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(512, 2) void paged_rows_kernel(PagedArgs p, float* ws, int parts) {
  constexpr int TK = kTileP, ROW = Lay<D>::ROW, GS = Lay<D>::GS, NG = 8 / GS, NM = D / 8, DB = D / 32, KS = D / 16, AHEAD = 6;
  constexpr int SLOT = TK * ROW;
  __shared__ u4 kbuf[4 * SLOT], vbuf[5 * SLOT];
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), behind = w >> 2;
  const int col = lane & 31, h = lane >> 5;
  const int kv = blockIdx.x % p.KVH, part = blockIdx.x / p.KVH % parts;
  int item = blockIdx.x / p.KVH / parts, seq = -1;
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
  if (__builtin_expect(seq < 0, 0)) {   // item: what is left of the block's number after all sequences' blocks
    if (part == 0) clear_unused<D, kRowsP>(kv, item);
    return;
  }

  const int r0 = item * kRowsP, total = sq.n * p.g, off = sq.len - sq.n;
  u4 q[KS];
  const Rows rw = load_rows<D>(p, sq, kv, r0 + 32 * w, q);
  have_queries(q);
  const int rl = r0 + kRowsP < total ? r0 + kRowsP - 1 : total - 1;
  const int first = uni(off + (int)p.gdiv.div(r0)), last = uni(off + (int)p.gdiv.div(rl));
  const PagedSpan span = paged_span(first, last, sq.len, sq.prefix, p.window, TK);
  // the part's tiles: begin .. begin + count
  const int all = uni(span.count()), per = tiles_per_part(all, parts, kPerMinP), begin = part * per;
  if (begin >= all && begin > 0) return;   // a row block that sees nothing is written by its first part
  const int count = all - begin < per ? all - begin : per;
  const bool whole = all <= per;
  auto tile_at = [&](int i) { return span.tile(begin + i); };

  // the wave's slots of a tile: 8 w .. 8 w + 8, in one page
  const Base kb = cache_base(p.k, kv), vb = cache_base(p.v, kv);
  uint32_t koff[NG], voff[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int j = GS * n + lane / ROW, piece = lane % ROW;
    koff[n] = j * kb.slot + 16u * (piece ^ Lay<D>::swz_k(8 * w + j));
    voff[n] = j * vb.slot + 16u * (piece ^ Lay<D>::swz_v(8 * w + j));
  }
  const int32_t* row = p.table + (int64_t)seq * p.ld_table;
  const int mask = (1 << p.shift) - 1;
  auto slot_of = [&](int i) { return tile_at(i < count ? i : count - 1) * TK + 8 * w; };
  int entries = 0;   // lane i: the table's entry for them in tile number i modulo 64
  // in steps, to be taken between MFMAs (past the last tile: zeros that nobody reads)
  struct {
    int j, n;
    uint32_t page, in;
    desc_t kd, vd;
  } ld;
  constexpr int LOAD_STEPS = 4 + NG;
  auto load_step = [&](int x, int i, int vslot) {
    if (x == 0) {
      ld.j = slot_of(i);
      const int id = __builtin_amdgcn_readlane(entries, i & 63);
      const bool ok = i < count && (uint32_t)id < (uint32_t)p.pages;
      ld.page = ok ? id : 0;
      ld.n = ok ? sq.len - ld.j : 0;
    } else if (x == 1) {
      ld.in = ld.j & mask;
      ld.n = ld.n < 0 ? 0 : (ld.n > 8 ? 8 : ld.n);
    } else if (x == 2) {
      ld.kd = make_desc(kb.at(ld.page, ld.in), ld.n * kb.slot);
    } else if (x == 3) {
      ld.vd = make_desc(vb.at(ld.page, ld.in), ld.n * vb.slot);
    } else {
      const int n = x - 4;
      lds_load16<true>(ld.kd, koff[n], kbuf + (i & 3) * SLOT + 64 * (NG * w + n));
      lds_load16<false>(ld.vd, voff[n], vbuf + vslot * SLOT + 64 * (NG * w + n));
    }
  };
  auto next_entries = [&](int i) {
    if ((i & 63) == 0 && i < count) {
      const int j = slot_of(i + lane);
      entries = row[(j < sq.len ? j : sq.len - 1) >> p.shift];
    }
  };
  auto load = [&](int i, int vslot) {
    next_entries(i);
#pragma unroll
    for (int x = 0; x < LOAD_STEPS; ++x) load_step(x, i, vslot);
  };
  // whether some page in reach is not one of the cache
  bool gaps = false;
  for (int range = 0; range < 2; ++range) {
    // the last tile may end past 2^31
    const int from = range ? span.lo * TK : 0, to = (int)min((int64_t)(range ? span.hi : span.pre) * TK, (int64_t)sq.len);
    for (int x = (from >> p.shift) + threadIdx.x; (int64_t)x << p.shift < to; x += 512) gaps |= row[x] < 0 || row[x] >= p.pages;
  }
  // values of "tile -1", which tile 0's first phase multiplies by weights of zero:
  // zeros themselves, as tile 0's own could be infinite (tile 4 takes their slot)
  for (int x = threadIdx.x; x < SLOT; x += 512) vbuf[4 * SLOT + x] = (u4){0u, 0u, 0u, 0u};
  gaps = uni(__syncthreads_or(gaps));
  auto exist = [&](int t0) -> uint64_t {   // bit per slot of a tile
    if (gaps) return __ballot(paged_page(row, t0 + lane, sq.len, p.shift, p.pages) >= 0);
    const int n = sq.len - t0;
    return n >= TK ? ~0ull : (1ull << n) - 1;
  };

  if (count > 0)
    for (int i = 0; i < 3; ++i) load(i, i);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // operands of MFMA m: keys (step m / 2, block m % 2), values (step m / DB, columns m % DB)
  const int kswz = Lay<D>::swz_k(col) ^ h, klow = col * ROW;
  const int li = lane & 15, key0 = 4 * h + (li >> 2), vlow = key0 * (D / 4) + (li & 1);
  const int vswz = Lay<D>::swz_v(key0) ^ (2 * ((lane >> 4) & 1) + ((li & 3) >> 1));
  auto key = [&](int t, int m) { return kbuf[(t & 3) * SLOT + klow + 32 * (m & 1) * ROW + (kswz ^ (2 * (m >> 1)))]; };
  auto value = [&](int vslot, int m) {
    const s4* a = (const s4*)(vbuf + vslot * SLOT) + vlow + 16 * (m / DB) * (D / 4) + 2 * ((4 * (m % DB)) ^ vswz);
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)a);
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(a + 8 * (D / 4)));
    return __builtin_bit_cast(u4, (s8v)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  Acc<D> ac;
  ac.clear();
  f16v s[2];
  uint32_t wt[16] = {};   // the tile's weights, two to a word; none before the first
  u4 frag[AHEAD];
  bool strange = false;   // some tile holds infinities or NaN that not every row sees
  const float c = __int_as_float(uni(__float_as_int(EXTRA ? 1.f : p.scale * kLog2e)));
  auto change = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // O += V P of the values in slot vs; frag: its first operands, on return the first of K in tile tk
  auto outputs = [&](int vs, int tk) {
    auto weight = [&](int m) {
      const int u = m / DB;
      return (u4){wt[4 * u], wt[4 * u + 1], wt[4 * u + 2], wt[4 * u + 3]};
    };
    // two at a time, the later operand first: one wait for both
#pragma unroll
    for (int m = 0; m < NM; m += 2) {
      T::add(ac.o[(m + 1) % DB], frag[(m + 1) % AHEAD], weight(m + 1));
      T::add(ac.o[m % DB], frag[m % AHEAD], weight(m));
#pragma unroll
      for (int x = m; x < m + 2; ++x) frag[x % AHEAD] = x + AHEAD < NM ? value(vs, x + AHEAD) : key(tk, (x + AHEAD) % NM);
      __builtin_amdgcn_sched_barrier(0);
    }
    u4 f[AHEAD];
#pragma unroll
    for (int m = 0; m < AHEAD; ++m) f[m] = frag[(m + NM) % AHEAD];
#pragma unroll
    for (int m = 0; m < AHEAD; ++m) frag[m] = f[m];
  };
  // S of tile t, and the loads of tile t + 3 between its products
  auto scores = [&](int t, int vslot) {
#pragma unroll
    for (int m = 0; m < NM; m += 2) {
      s[1] = T::mfma(frag[(m + 1) % AHEAD], q[m >> 1], m < 2 ? (f16v){} : s[1]);
      s[0] = T::mfma(frag[m % AHEAD], q[m >> 1], m < 2 ? (f16v){} : s[0]);
#pragma unroll
      for (int x = m; x < m + 2; ++x)
        if (x + AHEAD < NM) frag[x % AHEAD] = key(t, x + AHEAD);
#pragma unroll
      for (int x = m * LOAD_STEPS / NM; x < (m + 2) * LOAD_STEPS / NM; ++x) load_step(x, t + 3, vslot);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Weights of tile t.  No maximum beforehand: where a lane's 32 weights add up
  // to more than kMost (one may be too large for fp16, or the first tile has no
  // reference yet), the reference moves to kBelow under the largest score and
  // they are taken again, once.
  constexpr float kMost = 32768.f;
  // tiles [clean0, clean1) are seen whole by all the wave's rows
  int clean0 = count, clean1 = count;
  if (!gaps) {
    auto clean = [&](int i) {
      const int t0 = tile_at(i) * TK;
      return t0 + TK - 1 <= rw.first && t0 <= sq.len - TK && (p.window <= 0 || (int64_t)t0 > (int64_t)rw.last - p.window);
    };
    // one run of tiles: before it lie those of the prefix and the window's edge,
    // after it those past the wave's first row or the sequence
    while (clean1 > 0 && !clean(clean1 - 1)) --clean1;
    clean0 = 0;
    while (clean0 < clean1 && !clean(clean0)) ++clean0;
  }
  auto softmax = [&](int t, int vs) {
    if constexpr (EXTRA) cap_and_bias(p, rw, s, tile_at(t) * TK);
    if (t < clean0 || t >= clean1) {
      const int t0 = tile_at(t) * TK;
      hide(p, rw, sq, s, t0, exist(t0));
      strange |= not_finite<T>(vbuf + vs * SLOT, SLOT);
    }
    float l[2];
    auto weigh = [&] {
      const float nm = -ac.m;
      l[0] = l[1] = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k / 8][2 * (k % 8)], c, nm));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k / 8][2 * (k % 8) + 1], c, nm));
        l[0] += x;
        l[1] += y;
        wt[k] = pack2<T>(x, y);
      }
    };
    weigh();
    const float sum = l[0] + l[1];
    if (__builtin_expect(__any(sum > kMost), 0)) {
      float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int j = 1; j < 16; ++j) top = fmaxf(fmaxf(top, s[0][j]), s[1][j]);
      top = fmaxf(top, swap32(top)) * c;
      const float m2 = fmaxf(sum, swap32(sum)) > kMost ? top - kBelow : ac.m;
      const float f = __builtin_amdgcn_exp2f(ac.m - m2);
      ac.m = m2;
      ac.l[0] *= f;
      ac.l[1] *= f;
#pragma unroll
      for (int i = 0; i < DB; ++i) ac.o[i] *= f;
      weigh();
    }
    ac.l[0] += l[0];
    ac.l[1] += l[1];
#pragma unroll
    for (int k = 0; k < 16; ++k) asm volatile("" : "+v"(wt[k]));   // in this phase, not where they are used
#pragma unroll
    for (int m = 0; m < AHEAD; ++m) frag[m] = value(vs, m);   // landed long ago
  };

  change();
  if (behind) change();
#pragma unroll
  for (int m = 0; m < AHEAD; ++m) frag[m] = value(4, m);
  int vprev = 4, vcur = 0, vload = 3;   // slots of the values of tiles t - 1 (before tile 0: zeros), t, t + 3
#pragma unroll 1
  for (int t = 0; t < count; ++t) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NG) : "memory");   // tile t + 1 has landed; t + 2 may be on its way
    outputs(vprev, t);
    next_entries(t + 3);
    scores(t, vload);
    vload = vload == 4 ? 0 : vload + 1;
    change();
    softmax(t, vcur);
    vprev = vcur;
    vcur = vcur == 4 ? 0 : vcur + 1;
    change();
  }
  if (count > 0) outputs(vprev, count);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load into LDS outlives the workgroup
  if (!behind) change();
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");   // the last products have arrived
#pragma unroll
  for (int i = 0; i < DB; ++i) asm volatile("" : "+v"(ac.o[i]));
  Odd<D> odd;
  odd.clear();
  if (uni(__syncthreads_or(strange))) {
    // once more, a tile at a time, with what hides the hidden values
    ac.clear();
#pragma unroll 1
    for (int t = 0; t < count; ++t) {
      const int t0 = tile_at(t) * TK;
      load(t, 0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      tile<T, D, 2, EXTRA, true>(p, rw, sq, q, ac, odd, kbuf + (t & 3) * SLOT, vbuf, t0, exist(t0), [] {}, [] {});
      __syncthreads();
    }
  }

  const int r = r0 + 32 * w + col;
  const float l = ac.sum();
  if (r >= total) return;
  if (!whole) {
    float* rec = ws + (((int64_t)(blockIdx.x / p.KVH / parts) * p.KVH + kv) * parts + part) * record_floats(D, kRowsP);
    const int i = 32 * w + col;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = odd.fix(ac.o[db][4 * e + x], 16 * db + 4 * e + x);
        *(f4*)(rec + i * D + 32 * db + 8 * e + 4 * h) = v;
      }
    if (h == 0) {
      rec[kRowsP * D + 2 * i] = ac.m;
      rec[kRowsP * D + 2 * i + 1] = l;
    }
    return;
  }
  const float f = inverse(l);
  const int tok = (int)p.gdiv.div(r), a = kv * p.g + r - tok * p.g;
  const int64_t at = (int64_t)(sq.start + tok) * p.H + a;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f4 v;
#pragma unroll
      for (int x = 0; x < 4; ++x) v[x] = odd.fix(ac.o[db][4 * e + x] * f, 16 * db + 4 * e + x);
      store4<T>(p.out, at * D + 32 * db + 8 * e + 4 * h, v);
    }
  if (p.lse && h == 0) p.lse[at] = log_sum(ac.m, l);
}

// ---- few rows: one workgroup per 32 rows and a part of their tiles of 32 slots,
// which its four waves take in turn ----
//
// Reading the cache is all the work there is, so what counts is that many
// loads are on their way: 16 KiB per wave in one buffer for keys and one for
// values, each filled again as soon as its products have read it, two
// workgroups per CU.  Workgroups past a sequence's end return at once: the host
// does not know the lengths and launches for the longest that the table can
// hold.
//
// Measured (kernel, then join): four sequences of 90-131 thousand slots, 28 heads
// over 4, fp16, 961 MB: 172 + 10 us, 5.3 TB/s (a large copy 4.95; 191 with a
// wave to each part); 48 ragged sequences of up to 8000 slots, 191 MB: 42 + 5 us,
// bound by start-up and tail (124 with parts as long as the longest
// sequence asks for);
// one token behind 513 slots: 7.6 + 3.8, both mostly the launch (20.9 unsplit).

constexpr int kRowsS = 32, kTileS = 32;

// Row block `item` of the call: its sequence and number (-1: there is none; of
// chunks, how many blocks lie past the last).
__device__ __forceinline__ int find_block(const PagedArgs& p, int item, int rows, PagedSeq& sq, int& block) {
  if (!p.cu) {   // as many blocks for every sequence
    const int per = (p.g + rows - 1) / rows, s = uni(item / per);
    block = item - s * per;
    if (s >= p.b) return -1;
    const PagedSeq q = load_seq(p, s);
    sq = {uni(q.start), uni(q.n), uni(q.len), uni(q.prefix)};
    return block * rows < sq.n * p.g ? s : -1;
  }
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < p.b; s0 += 64) {
    const int s = s0 + lane;
    PagedSeq mine{};
    if (s < p.b) mine = load_seq(p, s);
    const int blocks = (int)(((int64_t)mine.n * p.g + rows - 1) / rows);
    int sum = blocks;   // at most rows * heads / 32 + b: an int
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(sum, o);
      if (lane >= o) sum += t;
    }
    const uint64_t past = __ballot(sum > item);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      sq.start = __builtin_amdgcn_readlane(mine.start, at);
      sq.n = __builtin_amdgcn_readlane(mine.n, at);
      sq.len = __builtin_amdgcn_readlane(mine.len, at);
      sq.prefix = __builtin_amdgcn_readlane(mine.prefix, at);
      block = item - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(blocks, at));
      return s0 + at;
    }
    item -= __builtin_amdgcn_readlane(sum, 63);
  }
  block = item;
  return -1;
}
__device__ __forceinline__ PagedSpan block_span(const PagedArgs& p, const PagedSeq& sq, int r0, int rows, int tk) {
  const int total = sq.n * p.g, off = sq.len - sq.n, rl = r0 + rows < total ? r0 + rows - 1 : total - 1;
  return paged_span(off + (int)p.gdiv.div(r0), off + (int)p.gdiv.div(rl), sq.len, sq.prefix, p.window, tk);
}

template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(256, 2) void paged_split_kernel(PagedArgs p, float* ws, int per_min, int R) {
  constexpr int TK = kTileS, ROW = Lay<D>::ROW, GS = Lay<D>::GS, NG = TK / GS;
  __shared__ u4 buf[4][2 * TK * ROW];   // a wave's keys, then values; its sums at the end
  __shared__ float ml[4][kRowsS][2];
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
  PagedSeq sq;
  int block;
  const int seq = find_block(p, blockIdx.z, kRowsS, sq, block), kv = blockIdx.y;
  if (__builtin_expect(seq < 0, 0)) {
    if (blockIdx.x == 0) clear_unused<D, kRowsS>(kv, block);
    return;
  }
  const int r0 = block * kRowsS, total = sq.n * p.g;
  const PagedSpan span = block_span(p, sq, r0, kRowsS, kTileS);
  const int count = uni(span.count()), per = tiles_per_part(count, gridDim.x, per_min), begin = blockIdx.x * per;
  if (begin >= count && begin > 0) return;   // a row block that sees nothing is written by its first part
  const int last = begin + per < count ? begin + per : count;
  const bool whole = count <= per;

  u4 *const kt = buf[w], *const vt = kt + TK * ROW;
  const int gl = lane / ROW, piece = lane % ROW, mask = (1 << p.shift) - 1;
  const Base kb = cache_base(p.k, kv), vb = cache_base(p.v, kv);
  uint32_t koff[D == 128 ? 4 : 2], voff[D == 128 ? 1 : 1];
#pragma unroll
  for (int n = 0; n < (D == 128 ? 4 : 2); ++n) koff[n] = gl * kb.slot + 16u * (piece ^ Lay<D>::swz_k(n * GS + gl));
  voff[0] = gl * vb.slot + 16u * (piece ^ Lay<D>::swz_v(gl));
  const int32_t* row = p.table + (int64_t)seq * p.ld_table;
  int base = 0, entries = 0;   // lane x: the table's entry for page number base + x of the sequence
  bool filled = false;
  struct {
    int t0, page[NG], n[NG];
    uint64_t vm;
  } nx;   // the tile that is loaded next
  auto look_up = [&](int i) {
    nx.t0 = span.tile(i) * TK;
    const int p0 = nx.t0 >> p.shift;
    if (!filled || p0 < base || ((nx.t0 + TK - 1) >> p.shift) >= base + 64) {
      filled = true;
      base = p0;
      const int top = (sq.len - 1) >> p.shift;   // a tile of the span begins before sq.len, or a page is not looked at
      entries = row[base + lane < top ? base + lane : top];
    }
    nx.vm = 0;
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      const int j = nx.t0 + gi * GS, id = __builtin_amdgcn_readlane(entries, (j >> p.shift) - base);
      const bool ok = j < sq.len && (uint32_t)id < (uint32_t)p.pages;
      nx.page[gi] = ok ? id : 0;
      nx.n[gi] = ok ? (sq.len - j < GS ? sq.len - j : GS) : 0;
      nx.vm |= (uint64_t)((1u << nx.n[gi]) - 1) << (gi * GS);
    }
  };
  auto load = [&](const Base& c, const uint32_t* off, int noff, u4* dst) {
#pragma unroll
    for (int gi = 0; gi < NG; ++gi)
      lds_load16(c.at(nx.page[gi], (nx.t0 + gi * GS) & mask), nx.n[gi] * c.slot, off[gi % noff], dst + 64 * gi);
  };
  constexpr int KO = D == 128 ? 4 : 2;
  u4 q[D / 16];
  const Rows rw = load_rows<D>(p, sq, kv, r0, q);
  int i = begin + w;
  if (i < last) look_up(i);
  have_queries(q);
  uint64_t vm = nx.vm;
  if (i < last) {
    load(kb, koff, KO, kt);
    load(vb, voff, 1, vt);
  }
  Acc<D> ac;
  ac.clear();
  Odd<D> odd;
  odd.clear();
#pragma unroll 1
  for (; i < last; i += 4) {
    // in order: keys i, values i, keys i + 4, values i + 4
    const int t0 = span.tile(i) * TK;
    const bool more = i + 4 < last;
    if (more) look_up(i + 4);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NG) : "memory");
    auto keys_done = [&] {   // the last of them read, whatever order the products were put in
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) load(kb, koff, KO, kt);
    };
    auto values_ready = [&] {
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NG) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    if (vm != 0xFFFFFFFFull || t0 + TK - 1 > rw.first || (p.window > 0 && (int64_t)t0 <= (int64_t)rw.last - p.window))
      tile<T, D, 1, EXTRA, true>(p, rw, sq, q, ac, odd, kt, vt, t0, vm, keys_done, values_ready);
    else
      tile<T, D, 1, EXTRA, false>(p, rw, sq, q, ac, odd, kt, vt, t0, vm, keys_done, values_ready);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the values are read
    if (more) load(vb, voff, 1, vt);
    vm = nx.vm;
  }

  // ---- the four waves' sums meet in LDS: piece d of row r (four outputs) at
  // [r][d ^ r], so that neither side meets a bank twice ----
  constexpr int P4 = D / 4;
  {
    const int r = lane & 31, h = lane >> 5;
    const float l = ac.sum();
    if (h == 0) {
      ml[w][r][0] = ac.m;
      ml[w][r][1] = l;
    }
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = odd.fix(ac.o[db][4 * e + x], 16 * db + 4 * e + x);
        ((f4*)kt)[r * P4 + ((db * 8 + 2 * e + h) ^ (r & (P4 - 1)))] = v;
      }
  }
  __syncthreads();
  float* rec = ws + (((int64_t)blockIdx.z * p.KVH + kv) * gridDim.x + blockIdx.x) * record_floats(D, R);
  const int d4 = tid % P4, rows = total - r0 < kRowsS ? total - r0 : kRowsS;
  for (int r = tid / P4; r < rows; r += 256 / P4) {
    float m = ml[0][r][0], l = 0.f;
#pragma unroll
    for (int x = 1; x < 4; ++x) m = fmaxf(m, ml[x][r][0]);
    f4 v = {};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = __builtin_amdgcn_exp2f(ml[x][r][0] - m);
      l += ml[x][r][1] * f;
      v += f * ((const f4*)buf[x])[r * P4 + (d4 ^ (r & (P4 - 1)))];
    }
    if (!whole) {
      *(f4*)(rec + r * D + 4 * d4) = v;
      if (d4 == 0) {
        rec[R * D + 2 * r] = m;
        rec[R * D + 2 * r + 1] = l;
      }
    } else {
      const int tok = (int)p.gdiv.div(r0 + r), a = kv * p.g + r0 + r - tok * p.g;
      const int64_t at = (int64_t)(sq.start + tok) * p.H + a;
      store4<T>(p.out, at * D + 4 * d4, v * inverse(l));
      if (p.lse && d4 == 0) p.lse[at] = log_sum(m, l);
    }
  }
}

// Adds up the parts of a row block, of 32 rows or (MANY) of 256.  SHARES = 1: a thread takes a piece of four
// outputs of its row through all parts, several rows to a workgroup; else each
// of SHARES threads takes every SHARES-th part, one row to a workgroup, and the
// shares are added up in their order.  16 shares take 10 us for the 128 parts of
// 28 heads and four long sequences; a call of one part has no join at all.
template <typename T, int D, int SHARES, bool MANY>
__global__ __launch_bounds__(SHARES == 1 ? 256 : D / 4 * SHARES) void paged_join_kernel(PagedArgs p, const float* ws, int parts_max,
                                                                                     int per_min, int R) {
  constexpr int P4 = D / 4;   // pieces of a row
  PagedSeq sq;
  int block;
  constexpr int ROWS = MANY ? kRowsP : kRowsS;
  const int seq = find_block(p, blockIdx.z, ROWS, sq, block), kv = blockIdx.y;
  if (seq < 0) return;
  if (MANY) block = (int)(((int64_t)sq.n * p.g + ROWS - 1) / ROWS) - 1 - block;   // that kernel takes the last rows first
  const int r0 = block * ROWS;
  const int count = block_span(p, sq, r0, ROWS, MANY ? kTileP : kTileS).count(), per = tiles_per_part(count, parts_max, per_min);
  const int parts = (count + per - 1) / per;
  const int d4 = threadIdx.x % P4, share = SHARES == 1 ? 0 : threadIdx.x / P4;
  const int r = SHARES == 1 ? blockIdx.x * (256 / P4) + threadIdx.x / P4 : blockIdx.x;
  if (parts <= 1) return;   // written by its only part
  const bool have = r < R && r0 + r < sq.n * p.g;
  if (!have && SHARES == 1) return;
  const float* base = ws + ((int64_t)blockIdx.z * p.KVH + kv) * parts_max * record_floats(D, R);
  float m = -3.0e38f, l = 0.f;
  f4 v = {};
  auto take = [&](float m1, float l1, f4 v1) {
    const float m2 = fmaxf(m, m1), f = __builtin_amdgcn_exp2f(m - m2), f1 = __builtin_amdgcn_exp2f(m1 - m2);
    m = m2;
    l = l * f + l1 * f1;
    v = v * f + v1 * f1;
  };
  if (have) {
#pragma unroll 8
    for (int x = share; x < parts; x += SHARES) {
      const float* rec = base + (int64_t)x * record_floats(D, R);
      take(rec[R * D + 2 * r], rec[R * D + 2 * r + 1], *(const f4*)(rec + r * D + 4 * d4));
    }
  }
  if constexpr (SHARES > 1) {
    __shared__ f4 part[SHARES][P4];
    __shared__ float pm[SHARES], pl[SHARES];
    part[share][d4] = v;
    if (d4 == 0) {
      pm[share] = m;
      pl[share] = l;
    }
    __syncthreads();
    if (share || !have) return;
    for (int x = 1; x < SHARES; ++x) take(pm[x], pl[x], part[x][d4]);
  }
  const int tok = (int)p.gdiv.div(r0 + r), a = kv * p.g + r0 + r - tok * p.g;
  const int64_t at = (int64_t)(sq.start + tok) * p.H + a;
  store4<T>(p.out, at * D + 4 * d4, v * inverse(l));
  if (p.lse && d4 == 0) p.lse[at] = log_sum(m, l);
}

// At most, over all sequences; with chunk offsets more than enough (clear_unused).
int64_t row_blocks(const PagedArgs& a, int rows) {
  return a.cu ? ((int64_t)a.rows * a.g + rows - 1) / rows + a.b : (int64_t)a.rows * ((a.g + rows - 1) / rows);
}
int64_t most_slots(const PagedArgs& a, int rows, int tk) {   // that a row block can see
  if (a.window > 0 && !a.prefix) return std::min<int64_t>(a.cap, (int64_t)a.window + rows + 2 * tk);
  return a.cap;
}
// Whether the sequences' chunks fill half a block of 256 rows on average, and
// there is work (rows by slots) enough for its longer start-up.  Single tokens
// never do: a block would hold the g rows of one (1280 tokens of 32 heads over 8,
// 500 slots: 1150 us, in blocks of 32 rows 440).  28 heads over 4, 128 wide, fp16, us
// in blocks of 32 rows and in blocks of 256 with their parts: 40 tokens over 600 slots
// (0.7 M) 15 and 27; 20 over 8192 (4.6 M) 33 and 32; 64 over 8192 57 and 38; 512 over
// 8192 189 and 77.  With a cap and a bias, whose softmax weighs more here: 4 chunks of
// 160 over 1000 slots (18 M) 63 and 67, 800 over 1000 (22 M) 66 and 67, 128 over 8192
// (29 M) 100 and 62; a bias alone would pay from less (800 over 1000: 62 and 50).  The
// average chunk decides, so a batch of single tokens and one chunk runs in one kind
// of block.
constexpr int64_t kWork = 4 << 20, kWorkExtra = 24 << 20;
bool many_rows(const PagedArgs& a) {
  const int64_t slots = a.window > 0 ? std::min<int64_t>(a.cap, (int64_t)a.window + kRowsP) : a.cap;
  return ((int64_t)(a.rows - a.b) * a.g >= 128 * (int64_t)a.b && (int64_t)a.rows * a.H * slots >= (a.extra() ? kWorkExtra : kWork)) ||
         row_blocks(a, kRowsS) > 65535;   // the grid's z
}
// The parts of a many-row call.  A workgroup takes a CU, so the time is rounds of
// workgroups: parts fill the chip where there are few row blocks and round off
// the last round where there are many.  Microseconds: 1.7 per tile of 128-wide
// heads, 6 until the first tile has landed, a part's record written and read
// again at the copy rate, 8 for the second launch; a tenth must be gained (4096
// tokens behind 28672 slots in four parts, 1.75 rounds for 2: 1690 us for 1665, the
// clock falls when all CUs work).  The time of a tile is that without caps and biases.
// 8192 slots, 28 heads over 4, blocks of 256 rows in one part and in these: 128 tokens
// 184 and 41 us, 512 184 and 77, 1100 185 and 139.
struct RowsPlan {
  int64_t blocks, parts;
  size_t ws_bytes;
};
RowsPlan rows_plan(const PagedArgs& a, int num_cus) {
  RowsPlan s;
  s.blocks = row_blocks(a, kRowsP);
  s.parts = 1;
  if (a.cu && s.blocks <= 65535) {
    const int64_t units = (((int64_t)a.rows * a.g + kRowsP - 1) / kRowsP + (a.b - 1) / 2) * a.KVH;   // half of each chunk's last block
    const int64_t tiles = (most_slots(a, kRowsP, kTileP) + kTileP - 1) / kTileP;
    const double record = (double)units * kRowsP * (a.D + 2) * sizeof(float) * 2 / 4.9e6, tile = 1.7 * a.D / 128;
    double least = 0;
    for (int parts = 1; parts <= 16 && (parts == 1 || parts * kPerMinP <= tiles); ++parts) {
      const int64_t rounds = (units * parts + num_cus - 1) / num_cus;
      const double t = (double)rounds * ((double)tiles / parts * tile + 6) + (parts > 1 ? 8 + parts * record : 0);
      if (parts == 1 || t < 0.9 * least) {
        least = t;
        s.parts = parts;
      }
    }
  }
  s.ws_bytes = s.parts > 1 ? (size_t)(s.blocks * a.KVH * s.parts) * record_floats(a.D, kRowsP) * sizeof(float) : 0;
  return s;
}

// The parts of a few-row call: as many for every row block, for sequences as
// long as the table (or the window) can hold; so many that the longest sequence
// of a ragged batch does not decide when the call ends, but of at least per_min
// tiles, more where there are row blocks enough to fill the chip.
struct SplitPlan {
  int64_t blocks, parts;
  int per_min, R;
  size_t ws_bytes;
};
SplitPlan split_plan(const PagedArgs& a, int num_cus) {
  SplitPlan s;
  s.blocks = row_blocks(a, kRowsS);
  const int64_t slots = most_slots(a, kRowsS, kTileS);
  const int64_t tiles = (slots + kTileS - 1) / kTileS, lanes = std::max<int64_t>(s.blocks * a.KVH, 1);
  s.per_min = lanes >= num_cus ? 16 : (4 * lanes >= num_cus ? 8 : 4);
  const int64_t want = std::max<int64_t>(1, (lanes >= num_cus ? 16 : 8) * (int64_t)num_cus / lanes);   // parts per row block and head
  s.parts = std::max<int64_t>(1, std::min(want, (tiles + s.per_min - 1) / s.per_min));
  const int64_t most = std::min<int64_t>(kRowsS, (a.cu ? (int64_t)a.rows : 1) * a.g);
  s.R = (int)((most + 7) / 8 * 8);
  s.ws_bytes = s.parts > 1 ? (size_t)(s.blocks * a.KVH * s.parts) * record_floats(a.D, s.R) * sizeof(float) : 0;
  return s;
}

template <typename T, int D>
hipError_t launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) {
  if (many_rows(a)) {
    const RowsPlan rp = rows_plan(a, num_cus);
    const int64_t grid = rp.blocks * a.KVH * rp.parts;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    if (a.extra()) paged_rows_kernel<T, D, true><<<(int)grid, 512, 0, s>>>(a, (float*)ws, (int)rp.parts);
    else paged_rows_kernel<T, D, false><<<(int)grid, 512, 0, s>>>(a, (float*)ws, (int)rp.parts);
    if (rp.parts > 1)
      paged_join_kernel<T, D, 1, true><<<dim3(kRowsP * D / 1024, a.KVH, (unsigned)rp.blocks), 256, 0, s>>>(a, (const float*)ws, (int)rp.parts, kPerMinP, kRowsP);
    return hipGetLastError();
  }
  const SplitPlan sp = split_plan(a, num_cus);
  const dim3 grid((unsigned)sp.parts, a.KVH, (unsigned)sp.blocks);
  if (a.extra()) paged_split_kernel<T, D, true><<<grid, 256, 0, s>>>(a, (float*)ws, sp.per_min, sp.R);
  else paged_split_kernel<T, D, false><<<grid, 256, 0, s>>>(a, (float*)ws, sp.per_min, sp.R);
  if (sp.parts > 16)
    paged_join_kernel<T, D, 16, false><<<dim3(sp.R, a.KVH, (unsigned)sp.blocks), D / 4 * 16, 0, s>>>(a, (const float*)ws, (int)sp.parts, sp.per_min, sp.R);
  else if (sp.parts > 1)
    paged_join_kernel<T, D, 1, false><<<dim3((sp.R + 1024 / D - 1) / (1024 / D), a.KVH, (unsigned)sp.blocks), 256, 0, s>>>(a, (const float*)ws, (int)sp.parts, sp.per_min, sp.R);
  return hipGetLastError();
}

}  // namespace

PagedPlan pattn_plan(const PagedArgs& a, int num_cus) {
  if (many_rows(a)) return {kRowsP, rows_plan(a, num_cus).parts};
  return {kRowsS, split_plan(a, num_cus).parts};
}

size_t pattn_workspace(const PagedArgs& a, int num_cus) {
  return many_rows(a) ? rows_plan(a, num_cus).ws_bytes : split_plan(a, num_cus).ws_bytes;
}

hipError_t pattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) {
  if (a.D == 128) return a.bf16 ? launch<BF16, 128>(a, num_cus, ws, s) : launch<F16, 128>(a, num_cus, ws, s);
  return a.bf16 ? launch<BF16, 64>(a, num_cus, ws, s) : launch<F16, 64>(a, num_cus, ws, s);
}

}  // namespace mq
