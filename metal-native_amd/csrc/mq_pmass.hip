// Attention weight that every cached key got:
//   mass[s][kv][j] = sum over the chunk's tokens and the query heads of kv of
//                    exp(x_rj - lse_r),
// x_rj the masked score of attention (mq_pattn.hip) and lse_r the log sum that
// attention left for the row, so a row's weights over its slots sum to one.  A
// row that saw nothing (lse -inf) adds nothing.
//
// A workgroup takes 256 slots, each wave 64 of them, whose keys stay in
// registers as the matrix instruction's second operand; the rows stream
// through LDS in blocks of 64, read once per workgroup.  With rows as the
// result's rows a lane's 16 results all belong to its own slot: the sum over
// rows needs no exchange but the last one between two lanes, and every output
// is written once, in a fixed order of additions.  Sums run over 16 rows, then
// 16 blocks, then all: fp32 throughout.
//
// Decode of 8 sequences of 2 to 16 thousand slots, 28 heads over 4, 54 MB of keys:
// 16.5 us (11 at the copy rate), bound by start-up and one wave of loads.  A chunk of
// 1500 tokens of each of two prompts of up to 8191 slots, bf16, 116 GFLOP: 258
// us, 0.45 PFLOP/s.  Per block of 64 rows a wave spends about 3000 cycles on 1024 of
// matrix work, the exponentials and the sums, and 1200 on the next block's loads and
// row data; eight waves per CU do not hide one another's.  Keeping the scores of
// one block in flight over the weights of the last gave 223 us but 22 for the
// decode (registers spilled), more parts 250 and 17.7: neither was kept.
#include "mq_paged_dev.hpp"

#include <algorithm>

namespace mq {
namespace {

constexpr int kSlotsM = 256, kRowsM = 64;

// The weight that slot j got from rows r0 .. r1 of sequence s's chunk, on all
// lanes of the wave: a row to a lane, in plain arithmetic, until it is NaN.  For
// slots whose sum above is NaN, which an infinite key makes of a row of zeros.
// The arguments (the kernel's first) are read once more from where they lie, so
// that none is kept in registers for this.
template <typename T, int D>
__device__ __forceinline__ float weight_of_slot(int s, int kv, int j, int r0, int64_t r1) {
  uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const PagedArgs& p = *(const PagedArgs*)args;
  const PagedSeq sq = load_seq(p, s);
  const int page = paged_page(p.table + (int64_t)s * p.ld_table, j, sq.len, p.shift, p.pages);
  if (page < 0) return 0.f;
  typedef typename T::e e8 __attribute__((ext_vector_type(8)));
  const e8* k = (const e8*)((const uint16_t*)p.k.ptr + page * p.k.page + kv * p.k.head + (int64_t)(j & ((1 << p.shift) - 1)) * p.k.slot);
  float t = 0.f;
#pragma unroll 1
  for (int64_t r = r0 + (int64_t)(threadIdx.x & 63); r < r1; r += 64) {
    const int i = (int)p.gdiv.div((uint32_t)r), a = kv * p.g + (int)r - i * p.g, pos = sq.len - sq.n + i;
    const float lse = p.lse[(int64_t)(sq.start + i) * p.H + a];
    const e8* q = (const e8*)((const uint16_t*)p.q + (int64_t)(sq.start + i) * p.q_t + (int64_t)a * p.q_h);
    float x = 0.f;
#pragma unroll 4
    for (int d = 0; d < D / 8; ++d) {
      const e8 y = q[d], z = k[d];
#pragma unroll
      for (int e = 0; e < 8; ++e) x += (float)y[e] * (float)z[e];
    }
    x *= p.scale;
    if (p.softcap != 0.f) x = p.softcap * (1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * p.inv_cap * (2.f * kLog2e)) + 1.f));
    if (p.slopes) x -= p.slopes[a] * fabsf((float)(pos - j));
    if (lse != -INFINITY && paged_visible(pos, j, sq.len, sq.prefix, p.window)) t += __builtin_amdgcn_exp2f((x - lse) * kLog2e);
    if (__any(t != t)) break;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
  return t;
}

template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(256, 2) void paged_mass_kernel(PagedArgs p, float* out, int parts) {
  constexpr int ROW = Lay<D>::ROW, GS = Lay<D>::GS, NG = kRowsM / GS / 4;
  __shared__ u4 qs[2][kRowsM * ROW];
  __shared__ float nl[2][kRowsM], sl[2][kRowsM];
  __shared__ int ps[2][kRowsM];
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), col = lane & 31, h = lane >> 5;
  const int slots = p.width << p.shift;
  const int part = blockIdx.x % parts, kv = (blockIdx.x / parts) % p.KVH, blk = blockIdx.x / parts / p.KVH, s = blockIdx.y;
  const PagedSeq sq0 = load_seq(p, s);
  const PagedSeq sq = {uni(sq0.start), uni(sq0.n), uni(sq0.len), uni(sq0.prefix)};
  const int j0 = blk * kSlotsM, off = sq.len - sq.n, total = sq.n * p.g;
  // rows that see a slot of the block, in blocks of kRowsM
  const PagedRange rr = paged_rows(j0, kSlotsM, sq, p.window, p.g);
  const int ra = rr.begin / kRowsM * kRowsM;
  const int blocks = rr.end > rr.begin ? (rr.end - ra - 1) / kRowsM + 1 : 0;
  const int b0 = (int)((int64_t)blocks * part / parts), b1 = (int)((int64_t)blocks * (part + 1) / parts);

  u4 kr[2][D / 16];
  bool have[2];
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int j = j0 + 64 * w + 32 * nb + col;
    const int page = b1 > b0 ? paged_page(p.table + (int64_t)s * p.ld_table, j, sq.len, p.shift, p.pages) : -1;
    have[nb] = page >= 0;
    const u4* src = (const u4*)((const uint16_t*)p.k.ptr + page * p.k.page + kv * p.k.head +
                                (int64_t)(j & ((1 << p.shift) - 1)) * p.k.slot) + h;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) kr[nb][ks] = have[nb] ? src[2 * ks] : (u4){0u, 0u, 0u, 0u};
  }

  const int gl = lane / ROW, piece = lane % ROW;
  auto load = [&](int b, u4* dst) {
    const int r0 = ra + b * kRowsM, tok0 = uni((int)p.gdiv.div(r0));
    const uint16_t* base = (const uint16_t*)p.q + (int64_t)(sq.start + tok0) * p.q_t + (int64_t)kv * p.g * p.q_h;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int gi = 4 * n + w, rl = gi * GS + gl, r = r0 + rl, i = (int)p.gdiv.div(r);
      const uint32_t off = 2u * ((uint32_t)(i - tok0) * (uint32_t)p.q_t + (uint32_t)(r - i * p.g) * (uint32_t)p.q_h) +
                           16u * (piece ^ Lay<D>::swz_k(rl));
      lds_load16(base, r0 + gi * GS < total ? 0x7fffffffu : 0u, r < total ? off : kOob, dst + 64 * gi);
    }
  };
  // lse of row `lane` of a block, and in wave 0 its position and slope
  float my_lse = 0.f, my_slope = 0.f;
  int my_pos = 0;
  auto row_info = [&](int b) {
    const int r = ra + b * kRowsM + lane;
    const int i = (int)p.gdiv.div(r), a = kv * p.g + r - i * p.g;
    my_pos = off + i;
    my_lse = r < total ? p.lse[(int64_t)(sq.start + i) * p.H + a] : -INFINITY;
    if (tid < kRowsM) my_slope = EXTRA && p.slopes && r < total ? p.slopes[a] : 0.f;
  };
  const int jw = j0 + 64 * w;
  float sum[2] = {0.f, 0.f}, mid[2] = {0.f, 0.f};
  auto step = [&](int b, int x) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (tid < kRowsM) {
      nl[x][tid] = my_lse == -INFINITY ? -INFINITY : -my_lse * kLog2e;
      ps[x][tid] = my_pos;
      sl[x][tid] = my_slope * kLog2e;
    }
    // rows of lse -inf add nothing, whatever their queries hold: each wave clears
    // those that it loaded (past the last row there are zeros already)
    const uint64_t none = __ballot(my_lse == -INFINITY && ra + b * kRowsM + lane < total);
    if (__builtin_expect(none != 0, 0)) {
      int l = lane;
      asm volatile("" : "+v"(l));   // nothing of this is kept over the blocks: it would cost a wave per SIMD
#pragma unroll 1
      for (int gi = w; gi < kRowsM / GS; gi += 4)
        if ((none >> (gi * GS + l / ROW)) & 1) qs[x][64 * gi + l] = (u4){0u, 0u, 0u, 0u};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (b + 1 < b1) {
      load(b + 1, qs[x ^ 1]);
      row_info(b + 1);
    }
    const int r0 = ra + b * kRowsM;
    const int first = off + (int)p.gdiv.div(r0), last = off + (int)p.gdiv.div(min(r0 + kRowsM, total) - 1);
    const bool masked = jw + 63 > first || (p.window > 0 && (int64_t)jw <= (int64_t)last - p.window);
#pragma unroll
    for (int rb2 = 0; rb2 < 2; ++rb2) {
      if (r0 + 32 * rb2 >= total) break;
      const int swz = Lay<D>::swz_k(col) ^ h;
      const u4* qt = qs[x] + (32 * rb2 + col) * ROW;
      f16v sc[2] = {};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const u4 a = qt[swz ^ (2 * ks)];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) sc[nb] = T::mfma(a, kr[nb][ks], sc[nb]);
      }
      float c = p.scale * kLog2e;
      if (EXTRA && p.softcap != 0.f) {
        cap_scores<false>(sc, p);   // a lane's are of 16 rows
        c = kLog2e;
      }
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        const int j = jw + 32 * nb + col;
        float t4[4];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int at = 32 * rb2 + 8 * q4 + 4 * h;
          const f4 n4 = *(const f4*)&nl[x][at];
          f4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float z = sc[nb][4 * q4 + e];
            if constexpr (EXTRA) z = z * c - sl[x][at + e] * fabsf((float)(ps[x][at + e] - j)) + n4[e];
            else z = __builtin_fmaf(z, c, n4[e]);
            v[e] = z;
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int pos = ps[x][at + e];
              const bool see = (j <= pos && (p.window <= 0 || (int64_t)j > (int64_t)pos - p.window)) || j < sq.prefix;
              v[e] = see ? v[e] : -INFINITY;
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_exp2f(v[e]);
          t4[q4] = (v[0] + v[1]) + (v[2] + v[3]);
        }
        mid[nb] += (t4[0] + t4[1]) + (t4[2] + t4[3]);
      }
    }
    if ((b & 15) == 15) {
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        sum[nb] += mid[nb];
        mid[nb] = 0.f;
      }
    }
  };
  if (b0 < b1) {
    load(b0, qs[b0 & 1]);
    row_info(b0);
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) asm volatile("" : "+v"(kr[nb][ks]));
    for (int b = b0; b < b1; ++b) step(b, b & 1);
  }
  float* dst = out + ((int64_t)part * p.b * p.KVH + (int64_t)s * p.KVH + kv) * slots;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    float t = sum[nb] + mid[nb];
    t += swap32(t);
    const int j = jw + 32 * nb + col;
    if (__builtin_expect(__any(t != t), 0)) {
      uint64_t again = __ballot(t != t) & 0xFFFFFFFFull;   // both halves hold t
      for (; again; again &= again - 1) {
        const int at = __ffsll((unsigned long long)again) - 1;
        const float v = weight_of_slot<T, D>(s, kv, jw + 32 * nb + at, ra + b0 * kRowsM, min(ra + (int64_t)b1 * kRowsM, (int64_t)total));
        if (col == at) t = v;
      }
    }
    if (h == 0 && j < slots) dst[j] = have[nb] ? t : 0.f;
  }
}

__global__ __launch_bounds__(256) void paged_mass_sum_kernel(const float* in, float* out, int64_t n, int parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float t = 0.f;
  for (int x = 0; x < parts; ++x) t += in[x * n + i];
  out[i] = t;
}

// Workgroups per 256 slots and key/value head: as many as bring the launch to
// two per CU, of at least four row blocks each.
int mass_parts(const PagedArgs& a, int num_cus) {
  const int64_t slots = (int64_t)a.width << a.shift;
  const int64_t wgs = (slots + kSlotsM - 1) / kSlotsM * a.KVH * a.b;
  const int64_t blocks = ((int64_t)a.max_q * a.g + kRowsM - 1) / kRowsM;
  return (int)std::max<int64_t>(1, std::min(2 * num_cus / std::max<int64_t>(wgs, 1), blocks / 4));
}

template <typename T, int D> hipError_t launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) {
  const int parts = mass_parts(a, num_cus);
  const int64_t slots = (int64_t)a.width << a.shift, n = slots * a.KVH * a.b;
  const int64_t gx = (slots + kSlotsM - 1) / kSlotsM * a.KVH * parts;
  if (gx > 0x7fffffff || a.b > 65535) return hipErrorInvalidValue;
  float* out = parts > 1 ? (float*)ws : a.mass;
  const dim3 grid((int)gx, a.b);
  if (a.extra()) paged_mass_kernel<T, D, true><<<grid, 256, 0, s>>>(a, out, parts);
  else paged_mass_kernel<T, D, false><<<grid, 256, 0, s>>>(a, out, parts);
  if (parts > 1) paged_mass_sum_kernel<<<(int)((n + 255) / 256), 256, 0, s>>>(out, a.mass, n, parts);
  return hipGetLastError();
}

}  // namespace

size_t pmass_workspace(const PagedArgs& a, int num_cus) {
  const int parts = mass_parts(a, num_cus);
  return parts > 1 ? sizeof(float) * parts * (((size_t)a.width << a.shift) * a.KVH * a.b) : 0;
}

hipError_t pmass_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s) {
  if (a.D == 128) return a.bf16 ? launch<BF16, 128>(a, num_cus, ws, s) : launch<F16, 128>(a, num_cus, ws, s);
  return a.bf16 ? launch<BF16, 64>(a, num_cus, ws, s) : launch<F16, 64>(a, num_cus, ws, s);
}

}  // namespace mq
