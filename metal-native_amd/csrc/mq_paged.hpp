// Paged key/value cache: arguments and addressing shared by the kernels that
// serve a model from it (mq_pattn.hip, mq_pmass.hip, mq_pcache.hip).
//
// A cache is [pages, kv_heads, page_size, head_dim] with unit stride along the
// last dimension; sequence s keeps slot j (the token at position j) in page
// table[s][j / page_size] at j % page_size.  Everything that says where a slot
// lies (lengths, chunk offsets, page numbers) is device memory that the host
// does not see, so every use of it here is bounded: lengths by the table's
// width, chunk offsets by the number of rows, and a slot whose page number is
// not a page of the cache counts as absent -- no kernel reads or writes it.
//
// The functions below that hold for host and device are the whole of that
// arithmetic; they build with a host compiler too.
#pragma once
#include <stdint.h>
#if defined(__HIP__) || defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define MQ_HD __host__ __device__ __forceinline__
#else
#define MQ_HD inline
#endif

namespace mq {

// One sequence of a call: its chunk's rows start .. start + n of the packed
// tokens, and its len cached slots (the chunk's own among them).
struct PagedSeq {
  int start, n, len, prefix;
};

// From the raw device values: cu (null: one row per sequence) may be anything,
// so a chunk is cut to the rows that exist; len to the slots that the table
// can name (cap); a prefix to the cached slots.
MQ_HD PagedSeq paged_seq(int s, int cu0, int cu1, bool has_cu, int len, int prefix, int rows, int cap) {
  PagedSeq r;
  if (!has_cu) {
    r.start = s;
    r.n = s < rows ? 1 : 0;
  } else {
    const int a = cu0 < 0 ? 0 : (cu0 > rows ? rows : cu0);
    const int b = cu1 < a ? a : (cu1 > rows ? rows : cu1);
    r.start = a;
    r.n = b - a;
  }
  r.len = len < 0 ? 0 : (len > cap ? cap : len);
  r.prefix = prefix < 0 ? 0 : (prefix > r.len ? r.len : prefix);
  return r;
}

// Key tiles of tk slots that the tokens at positions p0 .. p1 of a sequence
// can see: tiles [0, pre) of the prefix and [lo, hi) before the tokens, pre <=
// lo <= hi.  window <= 0: no window.  Tile number i of count() is tile(i).
struct PagedSpan {
  int pre, lo, hi;
  MQ_HD int count() const { return pre + hi - lo; }
  MQ_HD int tile(int i) const { return i < pre ? i : lo + (i - pre); }
};
MQ_HD PagedSpan paged_span(int p0, int p1, int len, int prefix, int window, int tk) {
  int end = p1 + 1 < len ? p1 + 1 : len;   // slots [0, end) but for the window
  if (end < 0) end = 0;
  int64_t first = window > 0 ? (int64_t)p0 - window + 1 : 0;
  if (first < 0) first = 0;
  PagedSpan s;
  s.hi = (int)(((int64_t)end + tk - 1) / tk);
  s.lo = (int)(first / tk);
  if (s.lo > s.hi) s.lo = s.hi;
  s.pre = (int)(((int64_t)prefix + tk - 1) / tk);   // prefix <= len
  if (s.pre >= s.lo) {   // the two ranges touch: one range from tile 0
    s.hi = s.pre > s.hi ? s.pre : s.hi;
    s.pre = 0;
    s.lo = 0;
  }
  return s;
}

MQ_HD bool paged_visible(int p, int j, int len, int prefix, int window) {
  return j >= 0 && j < len && ((j <= p && (window <= 0 || (int64_t)j > (int64_t)p - window)) || j < prefix);
}

// Rows of a sequence's chunk (g per token) whose tokens may see a slot of j0 ..
// j0 + slots - 1; none where the slots lie past the sequence.  Tokens are cut to
// the chunk's before they are multiplied: a table may name far more slots than
// the sequence has, and 2^31 rows' worth of them.
struct PagedRange {
  int begin, end;   // 0 <= begin <= end <= n * g
};
MQ_HD PagedRange paged_rows(int j0, int slots, const PagedSeq& s, int window, int g) {
  if (j0 >= s.len) return {0, 0};
  int64_t a = 0, b = s.n;
  if (j0 >= s.prefix) {
    const int64_t off = (int64_t)s.len - s.n;   // position of the chunk's first token
    a = (int64_t)j0 - off;
    a = a < 0 ? 0 : (a > s.n ? s.n : a);
    const int64_t end = (int64_t)j0 + slots - 1 + window - off;
    if (window > 0 && end < b) b = end;
  }
  return a < b ? PagedRange{(int)(a * g), (int)(b * g)} : PagedRange{0, 0};
}

// Bits d .. d + 63 of a row of `words` words; zeros outside them.
MQ_HD uint64_t paged_tree_bits(const uint64_t* row, int words, int64_t d) {
  if (d <= -64 || d >= (int64_t)words * 64) return 0;
  const int64_t w = d < 0 ? -1 : d >> 6;   // the word that holds bit d
  const int sh = (int)(d & 63);
  const uint64_t lo = w >= 0 ? row[w] >> sh : 0;
  const uint64_t hi = sh && w + 1 < words ? row[w + 1] << (64 - sh) : 0;
  return lo | hi;
}

// Whether some i, lo <= i <= hi for each of n terms, gives sum of step * i = rest:
// terms by falling steps (all positive), so that few i are left for each.  True too
// where `tries` does not settle it.
struct PagedTerm {
  int64_t step, lo, hi;
};
inline bool paged_reaches(const PagedTerm* t, int n, __int128 rest, int* tries) {
  if (n == 0) return rest == 0;
  __int128 lo = 0, hi = 0;   // what the other terms add
  for (int k = 1; k < n; ++k) {
    lo += (__int128)t[k].step * t[k].lo;
    hi += (__int128)t[k].step * t[k].hi;
  }
  const __int128 a = rest - hi, b = rest - lo, s = t[0].step;
  __int128 i = a >= 0 ? (a + s - 1) / s : -(-a / s), end = b >= 0 ? b / s : -((-b + s - 1) / s);
  if (i < t[0].lo) i = t[0].lo;
  if (end > t[0].hi) end = t[0].hi;
  for (; i <= end; ++i) {
    if (--*tries < 0 || paged_reaches(t + 1, n - 1, rest - s * i, tries)) return true;
  }
  return false;
}
// Whether two arrays of up to 8 dimensions of these sizes, with strides x and y, the
// second's first element `apart` elements behind the first's, may have one in common.
inline bool paged_share(int dims, const int64_t* size, const int64_t* x, const int64_t* y, int64_t apart) {
  PagedTerm t[16];
  int n = 0;
  auto add = [&](int64_t step, int64_t lo, int64_t hi) {
    if (step == 0 || lo == hi) return;
    int at = n++;
    for (; at > 0 && t[at - 1].step < step; --at) t[at] = t[at - 1];
    t[at] = {step, lo, hi};
  };
  for (int d = 0; d < dims; ++d) {
    const int64_t most = size[d] - 1;
    if (x[d] == y[d]) add(x[d], -most, most);
    else add(x[d], 0, most), add(y[d], -most, 0);
  }
  int tries = 4096;
  return paged_reaches(t, n, apart, &tries);
}

// Page that holds slot j, or -1 where there is none.
MQ_HD int paged_page(const int32_t* row, int j, int len, int shift, int pages) {
  if (j < 0 || j >= len) return -1;
  const int id = row[j >> shift];
  return id >= 0 && id < pages ? id : -1;
}

}  // namespace mq

#if defined(__HIP__) || defined(__HIPCC__)
#include "mq_launch.hpp"

namespace mq {

// Strides in elements; a slot is head_dim contiguous elements.
struct PagedCache {
  const void* ptr;
  int64_t page, head;
  int slot;
};

struct PagedArgs {
  const void* q;          // [rows, heads, dim], strides q_t, q_h
  int64_t q_t;
  int q_h;
  PagedCache k, v;
  const int32_t* table;   // [b, width], row stride ld_table
  int64_t ld_table;
  int width, pages, shift, cap;   // cap = min(width << shift, INT_MAX)
  const int32_t *lens, *cu, *prefix;
  const float* slopes;    // [heads] or null
  float scale, softcap;   // softcap 0: none
  float inv_cap;          // 1 / softcap, finite
  int window;             // 0: none
  int b, rows, H, KVH, g, D, bf16;
  int max_q;              // the longest chunk, as far as the host knows it
  Div32 gdiv;
  void* out;              // [rows, heads, dim] contiguous
  float* lse;             // [rows, heads] or null (attention); given (mass)
  float* mass;            // [b, kv_heads, width << shift]
  const uint64_t* tree;   // [rows, tree_words] ancestor bits of a tree's nodes, or null: a chunk in order
  int64_t ld_tree;
  int tree_words;
  bool extra() const { return softcap != 0.f || slopes != nullptr; }
};

struct PagedPlan {
  int block_rows;   // kRowsS or kRowsP of mq_pattn_dev.hpp
  int64_t parts;
};
PagedPlan pattn_plan(const PagedArgs& a, int num_cus);
size_t pattn_workspace(const PagedArgs& a, int num_cus);
hipError_t pattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s);
PagedPlan ptattn_plan(const PagedArgs& a, int num_cus);
size_t ptattn_workspace(const PagedArgs& a, int num_cus);
hipError_t ptattn_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s);   // a.tree set
size_t pmass_workspace(const PagedArgs& a, int num_cus);
hipError_t pmass_launch(const PagedArgs& a, int num_cus, void* ws, hipStream_t s);

struct PagedRopeArgs {
  const void* qkv;        // [rows, (H + 2 KVH) * D], row stride ld_qkv
  int64_t ld_qkv;
  const float *cos_t, *sin_t;   // [table_rows, D], row strides
  int64_t ld_cos, ld_sin;
  int64_t table_rows;
  const int64_t* pos;     // [axes, rows], axis stride ld_pos
  int64_t ld_pos;
  int axes, sec_end[8];   // frequencies [sec_end[a - 1], sec_end[a]) turn by axis a
  PagedCache k, v;
  const int32_t* table;
  int64_t ld_table;
  int width, pages, shift, cap;
  const int32_t *lens, *cu;
  int b, rows, H, KVH, D, bf16;
  void* q_out;            // [rows, H, D] contiguous
};
hipError_t prope_launch(const PagedRopeArgs& a, hipStream_t s);

struct PagedEvictArgs {
  PagedCache k, v;
  const int32_t* table;
  int64_t ld_table;
  int width, pages, shift, cap;
  const int32_t* lens;
  const float* mass;      // [b, KVH, slots], strides
  int64_t mass_b, mass_h;
  const int32_t* to;      // [b, to_width]
  int64_t ld_to;
  int to_width, budget, recent;
  int b, KVH, D;
  int32_t* kept;          // [b, KVH, budget]
  int32_t* new_lens;      // [b]
  float* left;            // [b, KVH, to_width << shift]
};
hipError_t pevict_launch(const PagedEvictArgs& a, int num_cus, hipStream_t s);

// A tree's nodes are the rows of its sequence's chunk; parents[row] is a node's
// number in it, smaller than the row's own, anything else no parent.
struct AncestorsArgs {
  const int32_t *parents, *cu;   // cu null: one row per sequence
  int b, rows, words;
  uint64_t* tree;   // [rows, words]
};
hipError_t pancestors_launch(const AncestorsArgs& a, hipStream_t s);

struct AcceptArgs {
  PagedCache k, v;
  int64_t k_layer, v_layer;   // strides of the caches' layers
  int layers;
  const int32_t* table;
  int64_t ld_table;
  int width, pages, shift, cap;
  const int32_t *lens, *cu;
  int b, rows, KVH, D, steps;
  const int64_t *drawn, *drafted;   // [rows]
  const int32_t* parents;           // [rows]
  int32_t *path, *count, *new_lens;   // [b, steps], [b], [b]
  int64_t* tokens;                    // [b, steps]
};
hipError_t paccept_launch(const AcceptArgs& a, hipStream_t s);

}  // namespace mq
#endif
