// C entries of the paged-cache operators: argument checks and launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdio>

#include "../../include/metal_native_amd.h"
#include "mq_paged.hpp"

namespace {

using mq::fail_with;

int log2_of(int64_t v) {
  int l = 0;
  while (((int64_t)1 << l) < v) ++l;
  return l;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// null, or what is wrong
const char* bad_cache(const mq_paged_cache* c, bool with_v) {
  if (!c || !c->k || (with_v && !c->v) || !c->table || !c->lens) return "null pointer in the cache";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
  if (c->dtype != MQ_PAGED_F16 && c->dtype != MQ_PAGED_BF16) return "unknown dtype";
  if (c->page_size < 8 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
    return "page_size must be a power of two from 8 to 65536";
  if (c->kv_heads < 1 || c->kv_heads > 65535 || c->pages < 1 || c->pages > INT_MAX || c->batch < 1 || c->batch > 65535 || c->width < 1)
    return "kv_heads and batch (at most 65535 each), pages and the table's width must be positive";
  if (c->width > INT_MAX / c->page_size) return "the table names 2^31 slots or more";
  if (c->batch > 1 && (c->ld_table < 0 || (c->width > 1 && c->ld_table < c->width))) return "the table's rows overlap";
  for (int i = 0; i < (with_v ? 2 : 1); ++i) {
    const int64_t page = i ? c->v_page : c->k_page, head = i ? c->v_head : c->k_head, slot = i ? c->v_slot : c->k_slot;
    if (!aligned16(i ? c->v : c->k) || page % 8 || head % 8 || slot % 8) return "the cache must be 16-byte aligned, its strides multiples of 8";
    if (slot < c->head_dim || slot > (1 << 26) || head < 0 || page < 0 || page >= (int64_t)1 << 31 ||
        (c->page_size - 1) * slot + c->head_dim >= (int64_t)1 << 31) return "strides of the cache out of range";
  }
  return nullptr;
}

int refuse(const char* op, const char* what) {
  char msg[256];
  std::snprintf(msg, sizeof msg, "%s: %s", op, what);
  return fail_with(MQ_INVALID_ARGUMENT, msg);
}

mq::PagedCache part(const void* p, int64_t page, int64_t head, int64_t slot) {
  mq::PagedCache c;
  c.ptr = p;
  c.page = page;
  c.head = head;
  c.slot = (int)slot;
  return c;
}

template <typename A> void fill_cache(A& a, const mq_paged_cache* c) {
  a.k = part(c->k, c->k_page, c->k_head, c->k_slot);
  a.v = part(c->v, c->v_page, c->v_head, c->v_slot);
  a.table = c->table;
  a.ld_table = c->ld_table;
  a.width = (int)c->width;
  a.pages = (int)c->pages;
  a.shift = log2_of(c->page_size);
  a.cap = (int)c->width << a.shift;
  a.lens = c->lens;
  a.b = (int)c->batch;
  a.KVH = c->kv_heads;
  a.D = c->head_dim;
}

// null, or what is wrong
const char* attn_args(mq::PagedArgs& a, const mq_paged_cache* c, const mq_paged_mask* m, int64_t rows, int32_t heads,
                      bool with_v) {
  if (const char* bad = bad_cache(c, with_v)) return bad;
  if (!m) return "null mask";
  if (rows < 0 || heads < 1 || heads % c->kv_heads) return "heads must be a multiple of kv_heads";
  if (rows > INT_MAX || rows * (int64_t)heads > INT_MAX) return "rows * heads must be below 2^31";
  if (!(m->scale > 0.f) || !std::isfinite(m->scale)) return "scale must be positive and finite";
  if (!(m->softcap >= 0.f) || !std::isfinite(m->softcap)) return "softcap must be zero or positive, and finite";
  if (m->window < 0) return "window must not be negative";
  if (!m->cu_q && rows != c->batch) return "without cu_q there must be one row per sequence";
  fill_cache(a, c);
  a.prefix = m->prefix_lens;
  a.cu = m->cu_q;
  a.slopes = m->slopes;
  a.scale = m->scale;
  a.softcap = m->softcap;
  a.inv_cap = m->softcap > 0.f ? std::min(1.f / m->softcap, FLT_MAX) : 0.f;
  a.window = m->window >= a.cap ? 0 : (int)m->window;   // as wide as any sequence: hides nothing
  a.rows = (int)rows;
  a.H = heads;
  a.g = heads / c->kv_heads;
  a.bf16 = c->dtype == MQ_PAGED_BF16;
  a.max_q = m->cu_q ? (int)(m->max_q < 1 || m->max_q > rows ? rows : m->max_q) : 1;
  a.gdiv = mq::Div32::make((uint32_t)a.g);
  a.q = nullptr;
  a.out = nullptr;
  a.lse = nullptr;
  a.mass = nullptr;
  return nullptr;
}

const char* query(mq::PagedArgs& a, const void* q, int64_t q_token, int64_t q_head) {
  if (!q) return "null queries";
  if (!aligned16(q) || q_token % 8 || q_head % 8 || q_token < 0 || q_head < 0)
    return "queries must be 16-byte aligned, their strides multiples of 8";
  // a block of rows is addressed by 32-bit offsets from its first token
  const int64_t most = (int64_t)1 << 29;
  if (q_token > most || q_head > most || a.g > 1 << 16 || 66 * q_token + a.g * q_head + a.D > most) return "strides of the queries out of range";
  a.q = q;
  a.q_t = q_token;
  a.q_h = (int)q_head;
  return nullptr;
}

}  // namespace

extern "C" {

MQ_API int mq_paged_rope_kv(const mq_paged_cache* c, const void* qkv, int64_t ld_qkv, const float* cos_t, int64_t ld_cos,
                            const float* sin_t, int64_t ld_sin, int64_t table_rows, const int64_t* pos, int64_t ld_pos,
                            int32_t axes, const int32_t* sections, const int32_t* cu_q, int64_t rows, int32_t heads,
                            void* q_out, void* stream) {
  const char* op = "paged.rope_kv";
  if (const char* bad = bad_cache(c, true)) return refuse(op, bad);
  if (!qkv || !cos_t || !sin_t || !pos || !q_out) return refuse(op, "null pointer argument");
  if (heads < 1 || heads % c->kv_heads) return refuse(op, "heads must be a multiple of kv_heads");
  const int64_t cols = ((int64_t)heads + 2 * c->kv_heads) * c->head_dim;
  if (cols > INT_MAX || rows < 0 || rows > INT_MAX) return refuse(op, "too many rows or heads");
  if (!cu_q && rows != c->batch) return refuse(op, "without cu_q there must be one row per sequence");
  if (!aligned16(qkv) || ld_qkv % 8 || (rows > 1 && ld_qkv < cols) || !aligned16(q_out))
    return refuse(op, "qkv rows must be 16-byte aligned");
  if (table_rows < 1 || !aligned16(cos_t) || !aligned16(sin_t) || ld_cos % 4 || ld_sin % 4 || ld_cos < 0 || ld_sin < 0)
    return refuse(op, "rotary tables must be 16-byte aligned and not empty");
  if (axes < 1 || axes > 8) return refuse(op, "one to eight axes");
  if (axes > 1 && ld_pos < 0) return refuse(op, "stride of the positions out of range");
  mq::PagedRopeArgs a{};
  int end = 0;
  for (int i = 0; i < 8; ++i) {
    if (i < axes) {
      const int n = sections ? sections[i] : c->head_dim / 2;
      if (n < 0 || n > c->head_dim / 2 || (!sections && axes > 1)) return refuse(op, "sections must be given, and not negative");
      end += n;
    }
    a.sec_end[i] = end;
  }
  if (end != c->head_dim / 2) return refuse(op, "sections must add up to head_dim / 2");
  fill_cache(a, c);
  a.qkv = qkv;
  a.ld_qkv = ld_qkv;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.ld_cos = ld_cos;
  a.ld_sin = ld_sin;
  a.table_rows = table_rows;
  a.pos = pos;
  a.ld_pos = ld_pos;
  a.axes = axes;
  a.cu = cu_q;
  a.rows = (int)rows;
  a.H = heads;
  a.bf16 = c->dtype == MQ_PAGED_BF16;
  a.q_out = q_out;
  const hipError_t e = mq::prope_launch(a, (hipStream_t)stream);
  return e == hipSuccess ? MQ_SUCCESS : mq::hip_fail_with(e, "paged.rope_kv: kernel launch failed");
}

MQ_API int64_t mq_paged_attention_workspace_size(const mq_paged_cache* c, const mq_paged_mask* m, int64_t rows,
                                                 int32_t heads) {
  mq::PagedArgs a;
  if (const char* bad = attn_args(a, c, m, rows, heads, true)) {
    refuse("paged.attention", bad);
    return -1;
  }
  return (int64_t)mq::pattn_workspace(a, mq::current_num_cus());
}

MQ_API int mq_paged_attention_plan(const mq_paged_cache* c, const mq_paged_mask* m, int64_t rows, int32_t heads,
                                   int32_t* block_rows, int32_t* parts) {
  const char* op = "paged.attention";
  mq::PagedArgs a;
  if (const char* bad = attn_args(a, c, m, rows, heads, true)) return refuse(op, bad);
  if (!block_rows || !parts) return refuse(op, "null output");
  const mq::PagedPlan plan = mq::pattn_plan(a, mq::current_num_cus());
  *block_rows = plan.block_rows;
  *parts = (int32_t)plan.parts;
  return MQ_SUCCESS;
}

MQ_API int mq_paged_attention(const mq_paged_cache* c, const mq_paged_mask* m, const void* q, int64_t q_token,
                              int64_t q_head, int64_t rows, int32_t heads, void* out, float* lse, void* ws,
                              int64_t ws_bytes, void* stream) {
  const char* op = "paged.attention";
  mq::PagedArgs a;
  if (const char* bad = attn_args(a, c, m, rows, heads, true)) return refuse(op, bad);
  if (rows == 0) return MQ_SUCCESS;
  if (const char* bad = query(a, q, q_token, q_head)) return refuse(op, bad);
  if (!out || !aligned16(out)) return refuse(op, "the output must be 16-byte aligned");
  a.out = out;
  a.lse = lse;
  const int cus = mq::current_num_cus();
  const size_t need = mq::pattn_workspace(a, cus);
  if (need && (!ws || !aligned16(ws) || ws_bytes < (int64_t)need)) return refuse(op, "workspace too small or not 16-byte aligned");
  const hipError_t e = mq::pattn_launch(a, cus, ws, (hipStream_t)stream);
  return e == hipSuccess ? MQ_SUCCESS : mq::hip_fail_with(e, "paged.attention: kernel launch failed");
}

MQ_API int64_t mq_paged_attention_mass_workspace_size(const mq_paged_cache* c, const mq_paged_mask* m, int64_t rows,
                                                      int32_t heads) {
  mq::PagedArgs a;
  if (const char* bad = attn_args(a, c, m, rows, heads, false)) {
    refuse("paged.attention_mass", bad);
    return -1;
  }
  return (int64_t)mq::pmass_workspace(a, mq::current_num_cus());
}

MQ_API int mq_paged_attention_mass(const mq_paged_cache* c, const mq_paged_mask* m, const void* q, int64_t q_token,
                                   int64_t q_head, int64_t rows, int32_t heads, const float* lse, float* mass, void* ws,
                                   int64_t ws_bytes, void* stream) {
  const char* op = "paged.attention_mass";
  mq::PagedArgs a;
  if (const char* bad = attn_args(a, c, m, rows, heads, false)) return refuse(op, bad);
  if (rows > 0) {
    if (const char* bad = query(a, q, q_token, q_head)) return refuse(op, bad);
    if (!lse) return refuse(op, "null lse");
  }
  if (!mass) return refuse(op, "null output");
  a.lse = const_cast<float*>(lse);
  a.mass = mass;
  const int cus = mq::current_num_cus();
  const size_t need = mq::pmass_workspace(a, cus);
  if (need && (!ws || ws_bytes < (int64_t)need)) return refuse(op, "workspace too small");
  const hipError_t e = mq::pmass_launch(a, cus, ws, (hipStream_t)stream);
  return e == hipSuccess ? MQ_SUCCESS : mq::hip_fail_with(e, "paged.attention_mass: kernel launch failed");
}

MQ_API int mq_paged_evict(const mq_paged_cache* c, const float* mass, int64_t mass_batch, int64_t mass_head,
                          const int32_t* to, int64_t ld_to, int64_t to_width, int64_t budget, int64_t recent,
                          int32_t* kept, int32_t* new_lens, float* left, void* stream) {
  const char* op = "paged.evict";
  if (const char* bad = bad_cache(c, true)) return refuse(op, bad);
  if (!mass || !to || !kept || !new_lens || !left) return refuse(op, "null pointer argument");
  if (budget < 1 || budget > INT_MAX || recent < 0 || recent > budget) return refuse(op, "recent must be 0 .. budget, budget positive");
  if (to_width < 1 || to_width > INT_MAX / c->page_size || to_width * c->page_size < budget)
    return refuse(op, "the target pages must hold the budget");
  if (mass_batch < 0 || mass_head < 0 || (c->batch > 1 && ld_to < to_width)) return refuse(op, "strides of mass or of the targets out of range");
  mq::PagedEvictArgs a{};
  fill_cache(a, c);
  a.mass = mass;
  a.mass_b = mass_batch;
  a.mass_h = mass_head;
  a.to = to;
  a.ld_to = ld_to;
  a.to_width = (int)to_width;
  a.budget = (int)budget;
  a.recent = (int)recent;
  a.kept = kept;
  a.new_lens = new_lens;
  a.left = left;
  const hipError_t e = mq::pevict_launch(a, mq::current_num_cus(), (hipStream_t)stream);
  return e == hipSuccess ? MQ_SUCCESS : mq::hip_fail_with(e, "paged.evict: kernel launch failed");
}

}  // extern "C"
