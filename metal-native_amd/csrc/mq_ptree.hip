// Trees of drafted tokens over a paged cache: ancestor bits, and the accepted
// path with its slots moved together.  Both are bound by latency: 64 trees of 100 to 512
// nodes are 1.2 MB, 48 paths of 28 layers and 4 heads of 128 move 5 MB (45 of 120 nodes
// change their slot: 1 us at the copy rate, the call takes 8.3).
#include "mq_paged_dev.hpp"

namespace mq {
namespace {

// A row's node and its ancestors as bits, by a walk from it to the root: parents have
// smaller numbers (anything else is no parent), so it ends, and words are written from
// the highest down.  i < 0: a row of no sequence.
__device__ __forceinline__ void walk(const AncestorsArgs& a, int row, int start, int i) {
  uint64_t* out = a.tree + (int64_t)row * a.words;
  uint64_t bits = 0;
  int w = a.words - 1;
  while (i >= 0) {
    const int at = i >> 6;
    for (; w > at; --w) {
      out[w] = bits;
      bits = 0;
    }
    if (at < a.words) bits |= 1ull << (i & 63);
    const int up = a.parents[start + i];
    i = up < i ? up : -1;
  }
  for (; w >= 0; --w) {
    out[w] = bits;
    bits = 0;
  }
}

// One token for each sequence: every row is a root.
__global__ __launch_bounds__(256) void roots_kernel(AncestorsArgs a) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row < a.rows) walk(a, row, row, 0);
}

// One workgroup per tree.  Trees of up to 512 nodes, one to a thread, by doubling: a
// node knows its ancestors up to some node, which knows its own up to another one, so
// 9 rounds take every path to its root.  Rows are written from LDS, their words in a row
// (64 trees of 100 to 512 nodes 6.9 us a call; each thread its own row 7.5; by walks
// through memory 13.8).  Larger trees, or rows of more words, go by these walks, a read
// behind another one for every ancestor: one tree of 1000 nodes 116 us, a chain 304, of
// 2500 643 and 1668.
constexpr int kNodes = 512, kNodeWords = kNodes / 64, kRounds = 10;
__global__ __launch_bounds__(kNodes) void ancestors_kernel(AncestorsArgs a) {
  __shared__ uint64_t bits[2][kNodeWords][kNodes];   // read and written in turn: one barrier a round
  __shared__ int ups[2][kNodes], goes_on[kRounds];
  const int s = blockIdx.x, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(s, a.cu[s], a.cu[s + 1], true, 0, 0, a.rows, 0);
  // rows before the first tree and past the last: no bits
  if (s == 0)
    for (int r = tid; r < min(a.cu[0], a.rows); r += kNodes) walk(a, r, r, -1);
  if (s == a.b - 1)
    for (int r = min(max(a.cu[a.b], 0), a.rows) + tid; r < a.rows; r += kNodes) walk(a, r, r, -1);
  if (sq.n > kNodes || a.words > kNodeWords) {
    for (int i = tid; i < sq.n; i += kNodes) walk(a, sq.start + i, sq.start, i);
    return;
  }
  const int words = min(a.words, (sq.n + 63) >> 6);   // those of the tree's own nodes; the others stay zero
  uint64_t mine[kNodeWords];
  int up = tid < sq.n ? a.parents[sq.start + tid] : -1;
  up = up < tid && up >= 0 ? up : -1;
#pragma unroll
  for (int w = 0; w < kNodeWords; ++w) {
    mine[w] = w == tid >> 6 ? 1ull << (tid & 63) : 0;
    if (w < words) bits[0][w][tid] = mine[w];
  }
  ups[0][tid] = up;
  if (tid < kRounds) goes_on[tid] = tid == 0;
  int round = 0;
  for (; round < kRounds - 1; ++round) {   // paths of up to 2^round nodes are whole
    __syncthreads();
    if (!goes_on[round]) break;
    const int from = round & 1, to = from ^ 1;
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < kNodeWords; ++w)
        if (w < words) mine[w] |= bits[from][w][up];
      up = ups[from][up];
    }
#pragma unroll
    for (int w = 0; w < kNodeWords; ++w)
      if (w < words) bits[to][w][tid] = mine[w];
    ups[to][tid] = up;
    if (up >= 0) goes_on[round + 1] = 1;
  }
  if (round == kRounds - 1) __syncthreads();
  uint64_t* out = a.tree + (int64_t)sq.start * a.words;
  for (int i = tid; i < sq.n * a.words; i += kNodes) {
    const int row = i / a.words, w = i - row * a.words;
    out[i] = w < words ? bits[round & 1][w][row] : 0;
  }
}

// A thread moves one 16-byte piece of a slot, of one layer, cache and head,
// through all of the path; every wave walks the path for itself.  Node i of the
// path goes to the i-th slot of the chunk, which is never behind its own: what a
// store overwrites is a slot that has been moved before, or by the same thread's
// loads in front of it.  Eight of a thread's loads are on their way at a time; every wave
// for itself needs no barrier and no second launch between the walk and the moves (one
// tree of 16 nodes 8.3 us a call, 4.0 of the kernel, 48 trees of 20 to 64 8.3 and 5.9).
__global__ __launch_bounds__(256) void accept_kernel(AcceptArgs a) {
  const int s = blockIdx.y, lane = threadIdx.x & 63;
  const PagedSeq sq = paged_seq(s, a.cu ? a.cu[s] : 0, a.cu ? a.cu[s + 1] : 0, a.cu != nullptr, a.lens[s], 0, a.rows, a.cap);
  const int off = sq.len - sq.n, per = a.D / 8, mask = (1 << a.shift) - 1;
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool have = x < (int64_t)a.layers * 2 * a.KVH * per;
  int64_t y = x / per;
  const int piece = (int)(x - y * per), head = (int)(y % a.KVH);
  y /= a.KVH;
  const PagedCache c = y & 1 ? a.v : a.k;
  u4* const base = (u4*)((uint16_t*)c.ptr + (y >> 1) * (y & 1 ? a.v_layer : a.k_layer) + head * c.head) + piece;
  const int32_t *row = a.table + (int64_t)s * a.ld_table, *parents = a.parents + sq.start;
  const int64_t *drawn = a.drawn + sq.start, *drafted = a.drafted + sq.start;
  const bool tells = blockIdx.x == 0 && threadIdx.x < 64;
  int cur = sq.n > 0 ? 0 : -1, done = 0;
  while (cur >= 0 && done < a.steps) {
    int mine = 0, m = 0;   // the path's next nodes: lane i the i-th
    while (cur >= 0 && m < 64 && done + m < a.steps) {
      if (lane == m) mine = cur;
      ++m;
      const int64_t want = drawn[cur];
      int next = -1;
      for (int i0 = cur + 1; i0 < sq.n && next < 0; i0 += 64) {
        const int i = i0 + lane;
        const uint64_t hit = __ballot(i < sq.n && parents[i] == cur && drafted[i] == want);
        if (hit) next = i0 + __ffsll((unsigned long long)hit) - 1;
      }
      cur = next;
    }
    if (tells && lane < m) {
      a.path[(int64_t)s * a.steps + done + lane] = mine;
      a.tokens[(int64_t)s * a.steps + done + lane] = drawn[mine];
    }
    const int from = off + mine, to = off + done + lane;
    const int page0 = lane < m && from != to ? paged_page(row, from, sq.len, a.shift, a.pages) : -1;
    const int page1 = page0 >= 0 ? paged_page(row, to, sq.len, a.shift, a.pages) : -1;
    for (int k0 = 0; k0 < m; k0 += 8) {
      u4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (__builtin_amdgcn_readlane(page1, k0 + k) >= 0 && have)
          v[k] = base[((int64_t)__builtin_amdgcn_readlane(page0, k0 + k) * c.page +
                       (int64_t)(__builtin_amdgcn_readlane(from, k0 + k) & mask) * c.slot) / 8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int page = __builtin_amdgcn_readlane(page1, k0 + k);
        if (page >= 0 && have) base[((int64_t)page * c.page + (int64_t)((off + done + k0 + k) & mask) * c.slot) / 8] = v[k];
      }
    }
    done += m;
  }
  if (!tells) return;
  for (int i = done + lane; i < a.steps; i += 64) {
    a.path[(int64_t)s * a.steps + i] = -1;
    a.tokens[(int64_t)s * a.steps + i] = -1;
  }
  if (lane == 0) {
    a.count[s] = done;
    a.new_lens[s] = max(off + done, 0);
  }
}

}  // namespace

hipError_t pancestors_launch(const AncestorsArgs& a, hipStream_t s) {
  if (a.cu) ancestors_kernel<<<a.b, kNodes, 0, s>>>(a);
  else roots_kernel<<<(a.rows + 255) / 256, 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t paccept_launch(const AcceptArgs& a, hipStream_t s) {
  const int64_t pieces = (int64_t)a.layers * 2 * a.KVH * (a.D / 8);
  const int64_t blocks = (pieces + 255) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  accept_kernel<<<dim3((unsigned)blocks, a.b), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace mq
