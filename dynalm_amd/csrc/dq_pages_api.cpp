// dq_pages_api.cpp -- the long caches' C ABI (declared in include/dynaq.h): argument checks with
// dynacore's status codes, then the launches. Nothing is allocated or kept.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/dynaq.h"
#include "dq_attn.h"
#include "dq_attn_checks.h"
#include "dq_internal.h"
#include "dq_pages.h"

namespace {

using namespace dq;

constexpr int64_t kMostKeys = (int64_t)1 << 29;  // keys of a sequence, entries of a list
constexpr int64_t kWorkspace = DQ_ATTENTION_WORKSPACE_BYTES;

int too_many(const char* what) { return set_error(DQ_UNSUPPORTED, "%s are too many for a launch", what); }

// The batch and its keys; page_size 0: without their pages.
int check_sequences(const dq_sequences* s, int64_t page_size) {
  if (s == nullptr) return bad("sequences: null argument");
  if (s->batch < 0 || s->batch > INT32_MAX / 2) return set_error(DQ_INVALID_ARGUMENT, "batch %lld", (ll)s->batch);
  if (s->max_len < 0 || s->max_len > kMostKeys) return set_error(DQ_INVALID_ARGUMENT, "max_len %lld: 0..2^29 keys", (ll)s->max_len);
  if (page_size > 0 && (s->pages_stride < ceil_div(s->max_len, page_size) || s->pages_stride > kMostKeys))
    return set_error(DQ_INVALID_ARGUMENT, "pages_stride %lld: max_len %lld needs %lld pages", (ll)s->pages_stride, (ll)s->max_len,
                     (ll)ceil_div(s->max_len, page_size));
  return DQ_OK;
}

int check_sequence_data(const dq_sequences* s, const dq_kv_cache* c) {
  if (s->batch == 0 || s->max_len == 0) return DQ_OK;
  if (s->lens == nullptr) return bad("lens: null argument");
  if (c != nullptr && s->pages == nullptr) return bad("pages: null argument");
  if (c != nullptr && c->n_pages == 0) return bad("cache: no pages");
  return DQ_OK;
}

// The rows of the sequences and their query heads.
int check_queries(const dq_kv_cache* c, const dq_sequences* s, const dq_heads* q, bool data) {
  if (s->tokens < 0) return bad("tokens must be >= 0");
  if (s->max_q < 1) return set_error(DQ_INVALID_ARGUMENT, "max_q %lld", (ll)s->max_q);
  if (int rc = check_rows("q", q, s->tokens); rc != DQ_OK) return rc;
  if (q->dtype != DQ_F32 && q->dtype != c->dtype)
    return set_error(DQ_UNSUPPORTED, "q type %d with cache type %d: q has the cache's type or fp32", q->dtype, c->dtype);
  if (q->heads % c->kv_heads != 0) return set_error(DQ_INVALID_ARGUMENT, "%d query heads, %d kv heads", q->heads, c->kv_heads);
  // (head rows are counted in 32 bits)
  if (s->tokens > ((int64_t)1 << 30) / q->heads)
    return set_error(DQ_UNSUPPORTED, "%lld tokens of %d heads are too many", (ll)s->tokens, q->heads);
  if (data && s->q_offsets == nullptr && (s->tokens != s->batch || s->max_q != 1))
    return bad("without q_offsets every sequence has one token");
  return DQ_OK;
}

// A cache whose keys alone are read (its values too where `values`).
int check_read(const dq_kv_cache* c, bool values) {
  if (c->n_pages == 0) return DQ_OK;
  if (c->k == nullptr || (values && c->v == nullptr)) return bad("cache: null pointer");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(values ? c->v : nullptr)) % 16 != 0)
    return bad("cache: k and v must be 16-byte aligned");
  return DQ_OK;
}

// Keys are addressed from their page in 32 bits.
int check_token_stride(const dq_kv_cache* c) {
  if (c->token_stride > (1 << 25)) return set_error(DQ_UNSUPPORTED, "cache: token_stride %lld", (ll)c->token_stride);
  return DQ_OK;
}

int check_scale(float scale) {
  if (!(scale > 0) || !std::isfinite(scale * kLog2e)) return bad("scale must be positive and finite");
  return DQ_OK;
}

// Weights of the sequences' heads, apart from each other.
int check_mass(const float* mass, const dq_sequences* s, int64_t heads, int64_t seq, int64_t head) {
  if (seq < 0 || head < 0 || seq > ((int64_t)1 << 58) / (s->batch + 1) || head > ((int64_t)1 << 58) / heads)
    return bad("mass: strides are negative or too large");
  // (the axis of shorter strides, within the other)
  const bool heads_far = s->batch > 1 && (heads == 1 || seq < head);
  const int64_t n = heads_far ? s->batch : heads, step = heads_far ? seq : head;
  const int64_t far_n = heads_far ? heads : s->batch, far = heads_far ? head : seq;
  if ((n > 1 && step < s->max_len) || (far_n > 1 && far < (n - 1) * step + s->max_len))
    return set_error(DQ_INVALID_ARGUMENT, "mass: rows overlap (seq_stride %lld, head_stride %lld)", (ll)seq, (ll)head);
  if (s->batch > 0 && s->max_len > 0) {
    if (mass == nullptr) return bad("mass: null argument");
    if (reinterpret_cast<uintptr_t>(mass) % 4 != 0) return bad("mass: misaligned pointer");
  }
  return DQ_OK;
}

int check_workspace(const void* p, int64_t bytes, int64_t need) {
  if (need == 0) return DQ_OK;
  if (p == nullptr) return bad("workspace: null argument");
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return bad("workspace: must be 16-byte aligned");
  if (bytes < need) return set_error(DQ_RESOURCE_EXHAUSTED, "workspace: %lld bytes, the call needs %lld", (ll)bytes, (ll)need);
  return DQ_OK;
}

AttnArgs sequence_args(const dq_kv_cache* c, const dq_sequences* s) {
  AttnArgs r;
  r.cache = cache_args(c);
  r.dim = c->head_dim;
  r.batch = (int32_t)s->batch;
  r.q_offsets = s->q_offsets;
  r.pages = s->pages;
  r.pages_stride = s->pages_stride;
  r.lens = s->lens;
  r.max_len = (int32_t)s->max_len;
  return r;
}

AttnArgs query_args(const dq_kv_cache* c, const dq_sequences* s, const dq_heads* q, float scale) {
  AttnArgs r = sequence_args(c, s);
  r.tokens = r.part_tokens = (int32_t)s->tokens;
  r.max_q = (int32_t)std::min(s->max_q, s->tokens);
  r.q = q->p;
  r.q_token = q->token_stride;
  r.q_head = q->head_stride;
  r.q_vec = aligned(q, 16);
  r.heads = q->heads;
  r.group = q->heads / c->kv_heads;
  r.scale_log2 = std::fmax(scale * kLog2e, 1.2e-38f);
  return r;
}

// ---- plans: functions of the shape ----

// Tokens whose scores a launch of dq_choose_pages writes (0: one's are too many).
int64_t choose_tokens(const dq_kv_cache* c, const dq_sequences* s, bool scores) {
  const int64_t pages = ceil_div(s->max_len, c->page_size);
  int64_t n = (kMaxGroups / 4 - 1) / c->kv_heads;  // (a workgroup of 1,024 threads a row at most)
  if (scores) n = std::min(n, kWorkspace / 8 / pages / c->kv_heads);
  return std::min(n, s->tokens);
}

int check_choose(const dq_kv_cache* c, const dq_sequences* s) {
  if (int rc = check_cache(c, false); rc != DQ_OK) return rc;
  if (int rc = check_sequences(s, c->page_size); rc != DQ_OK) return rc;
  if (s->tokens < 0) return bad("tokens must be >= 0");
  if (s->tokens > 0 && s->max_len > 0 &&
      (choose_tokens(c, s, true) == 0 || s->batch > (kMaxGroups - 1) / (ceil_div(ceil_div(s->max_len, c->page_size), 64) * c->kv_heads)))
    return too_many("pages and heads");
  return DQ_OK;
}

struct PagePlan {
  int64_t splits = 1, chunk = 0, items = 0;
  int64_t bytes = 0;
};

// Items that a launch of dq_page_attention aims at, one a CU, and keys that are worth one. 256 / 512 / 1,024 items, us, 8 kv heads of 128: 4
// sequences of 4,096 keys 18.5 / 19.5 / 19.8, 16: 45.9 / 46.3 / 47.0, 32: 105.7 / 108.0 / 110.9; 32 of 1,024 keys 24.1 / 28.0 / 28.8.
constexpr int64_t kPageItems = 256, kPageKeys = 256;

PagePlan plan_pages(const dq_kv_cache* c, const dq_sequences* s, const dq_heads* q, int64_t count) {
  PagePlan p;
  const int64_t group = q->heads / c->kv_heads, rows = s->tokens * c->kv_heads * ceil_div(group, 16);
  const int64_t keys = std::min(std::min(count, ceil_div(s->max_len, c->page_size)) * c->page_size, s->max_len);
  if (rows > 0) p.splits = std::max<int64_t>(1, std::min(kPageItems / rows, keys / kPageKeys));
  p.chunk = std::max<int64_t>(1, ceil_div(count, p.splits));
  p.splits = std::max<int64_t>(1, ceil_div(count, p.chunk));
  p.items = rows * p.splits;
  if (p.splits > 1) p.bytes = p.splits * s->tokens * q->heads * (c->head_dim + 2) * 4;
  return p;
}

int check_page_attention(const dq_kv_cache* c, const dq_sequences* s, const dq_heads* q, int64_t count, bool data) {
  if (int rc = check_cache(c, data); rc != DQ_OK) return rc;
  if (int rc = check_token_stride(c); rc != DQ_OK) return rc;
  if (int rc = check_sequences(s, c->page_size); rc != DQ_OK) return rc;
  if (int rc = check_queries(c, s, q, data); rc != DQ_OK) return rc;
  if (c->page_size > (1 << 24)) return set_error(DQ_UNSUPPORTED, "cache: page_size %d", c->page_size);  // (64 pages' keys are counted in 32 bits)
  if (count < 1 || count > kMostKeys) return set_error(DQ_INVALID_ARGUMENT, "count %lld", (ll)count);
  if (plan_pages(c, s, q, count).items >= kMaxGroups) return too_many("rows");
  return DQ_OK;
}

struct MassPlan {
  int64_t splits = 1, items = 0;
  int64_t bytes = 0;
};

// Items that a launch of dq_attention_mass aims at (768 / 1,024 / 1,536 / 2,048: 104 / 96 / 93 / 92 us and 4.8 / 5.1 / 6.2 / 7.3 for the join), keys of one, and rows that are worth one: fewer where items are so few that CUs
// would be idle: 10 items of 352 fp32 rows in heads of 256, us with and without: 21 and 47; 18 items of 1,336 rows 14.8 and 18.5; at 512 items
// in place of 256: 14 sequences of 128 rows 29 in place of 17.
constexpr int64_t kMassItems = 1536, kMassKeys = 256, kMassRows = 256;
constexpr int64_t kMassFewItems = 256, kMassFewRows = 64;

MassPlan plan_mass(const dq_kv_cache* c, const dq_sequences* s, const dq_heads* q) {
  MassPlan p;
  const int64_t rows = std::min(s->max_q, s->tokens) * (q->heads / c->kv_heads);
  const int64_t items = s->batch * c->kv_heads * ceil_div(s->max_len, kMassKeys), keys = s->batch * c->kv_heads * s->max_len * 4;
  if (items > 0) {
    p.splits = std::max(std::min(kMassItems / items, rows / kMassRows), std::min(kMassFewItems / items, rows / kMassFewRows));
    p.splits = std::max<int64_t>(1, std::min(p.splits, kWorkspace / keys));
  }
  p.items = items * p.splits;
  if (p.splits > 1) p.bytes = p.splits * keys;
  return p;
}

int check_mass_call(const dq_kv_cache* c, const dq_sequences* s, const dq_heads* q, bool data) {
  if (int rc = check_cache(c, false); rc != DQ_OK) return rc;
  if (int rc = check_token_stride(c); rc != DQ_OK) return rc;
  if (int rc = check_sequences(s, c->page_size); rc != DQ_OK) return rc;
  if (int rc = check_queries(c, s, q, data); rc != DQ_OK) return rc;
  if (s->batch * ceil_div(s->max_len, kMassKeys) >= kMaxGroups / c->kv_heads) return too_many("keys");
  return DQ_OK;
}

}  // namespace

extern "C" {

int dq_page_bounds(const dq_kv_cache* cache, const dq_sequences* s, const int32_t* from, int64_t max_new, void* bounds,
                   void* stream) {
  if (int rc = check_cache(cache, false); rc != DQ_OK) return rc;
  if (int rc = check_sequences(s, cache->page_size); rc != DQ_OK) return rc;
  if (from != nullptr && max_new < 0) return bad("max_new must be >= 0");
  if (s->batch == 0 || s->max_len == 0 || (from != nullptr && max_new == 0)) return DQ_OK;
  if (int rc = check_sequence_data(s, cache); rc != DQ_OK) return rc;
  if (int rc = check_read(cache, false); rc != DQ_OK) return rc;
  if (bounds == nullptr) return bad("bounds: null argument");
  if (reinterpret_cast<uintptr_t>(bounds) % 16 != 0) return bad("bounds: must be 16-byte aligned");
  const int64_t all = ceil_div(s->max_len, cache->page_size);
  const int64_t slots = from == nullptr ? all : std::min(all, ceil_div(std::min(max_new, s->max_len), cache->page_size) + 1);
  if (slots > ((int64_t)1 << 60) / s->batch / cache->kv_heads) return too_many("pages");
  const hipError_t e = launch_page_bounds(cache->dtype, sequence_args(cache, s), from, slots, static_cast<uint16_t*>(bounds),
                                          static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "page_bounds launch");
}

int64_t dq_choose_pages_workspace(const dq_kv_cache* cache, const dq_sequences* s) {
  if (int rc = check_choose(cache, s); rc != DQ_OK) return -rc;
  if (s->tokens == 0 || s->max_len == 0) return 0;
  return choose_tokens(cache, s, true) * cache->kv_heads * ceil_div(s->max_len, cache->page_size) * 8;
}

int dq_choose_pages(const dq_kv_cache* cache, const dq_sequences* s, const dq_heads* q, const void* bounds, int64_t first,
                    int64_t last, int64_t count, int32_t* chosen, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_choose(cache, s); rc != DQ_OK) return rc;
  if (int rc = check_queries(cache, s, q, true); rc != DQ_OK) return rc;
  if (count < 1 || count > kMostKeys) return set_error(DQ_INVALID_ARGUMENT, "count %lld", (ll)count);
  if (first < 0 || last < 1 || first > count || last > count - first)
    return set_error(DQ_INVALID_ARGUMENT, "first %lld and last %lld of %lld pages: last is 1 or more, their sum at most count", (ll)first,
                     (ll)last, (ll)count);
  if (s->tokens == 0 || s->batch == 0) return DQ_OK;
  if (int rc = check_sequence_data(s, cache); rc != DQ_OK) return rc;
  if (int rc = check_data("q", q); rc != DQ_OK) return rc;
  if (chosen == nullptr) return bad("chosen: null argument");
  const int64_t pages = ceil_div(s->max_len, cache->page_size);
  const bool scores = pages > count;
  ChooseArgs c;
  c.chosen = chosen;
  c.pages = (int32_t)pages;
  c.first = (int32_t)first;
  c.last = (int32_t)last;
  c.count = count;
  c.tokens = choose_tokens(cache, s, scores);
  if (c.tokens == 0) return too_many("heads");
  if (scores) {
    if (bounds == nullptr) return bad("bounds: null argument");
    if (reinterpret_cast<uintptr_t>(bounds) % 16 != 0) return bad("bounds: must be 16-byte aligned");
    if (int rc = check_workspace(workspace, workspace_bytes, c.tokens * cache->kv_heads * pages * 8); rc != DQ_OK) return rc;
    c.bounds = static_cast<const uint16_t*>(bounds);
    c.keys = static_cast<uint64_t*>(workspace);
  }
  const hipError_t e = launch_choose_pages(q->dtype, cache->dtype, query_args(cache, s, q, 1.f), c, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "choose_pages launch");
}

int64_t dq_page_attention_workspace(const dq_kv_cache* cache, const dq_sequences* s, const dq_heads* q, int64_t count) {
  if (int rc = check_page_attention(cache, s, q, count, false); rc != DQ_OK) return -rc;
  return plan_pages(cache, s, q, count).bytes;
}

int dq_page_attention(const dq_kv_cache* cache, const dq_sequences* s, const dq_heads* q, const dq_heads* out, float* lse,
                      const int32_t* chosen, int64_t count, float scale, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  if (int rc = check_page_attention(cache, s, q, count, true); rc != DQ_OK) return rc;
  if (int rc = check_rows("out", out, s->tokens); rc != DQ_OK) return rc;
  if (int rc = check_apart("out", out, s->tokens, cache->head_dim); rc != DQ_OK) return rc;
  if (out->dtype != q->dtype) return set_error(DQ_UNSUPPORTED, "q and out differ in type");
  if (out->heads != q->heads) return set_error(DQ_INVALID_ARGUMENT, "%d query heads, %d of out", q->heads, out->heads);
  if (int rc = check_scale(scale); rc != DQ_OK) return rc;
  if (s->tokens == 0 || s->batch == 0) return DQ_OK;
  if (int rc = check_sequence_data(s, cache); rc != DQ_OK) return rc;
  if (int rc = check_data("q", q); rc != DQ_OK) return rc;
  if (int rc = check_data("out", out); rc != DQ_OK) return rc;
  if (chosen == nullptr) return bad("chosen: null argument");
  const PagePlan p = plan_pages(cache, s, q, count);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes); rc != DQ_OK) return rc;
  AttnArgs a = query_args(cache, s, q, scale);
  a.out = out->p;
  a.out_token = out->token_stride;
  a.out_head = out->head_stride;
  a.out_vec = aligned(out, 4 * float_bytes(out->dtype));
  a.lse = lse;
  if (p.splits > 1) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + p.splits * s->tokens * q->heads * cache->head_dim;
  }
  const hipError_t e = launch_page_attention(q->dtype, cache->dtype, a, chosen, count, (int32_t)p.splits, (int32_t)p.chunk,
                                             static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "page_attention launch");
}

int64_t dq_attention_mass_workspace(const dq_kv_cache* cache, const dq_sequences* s, const dq_heads* q) {
  if (int rc = check_mass_call(cache, s, q, false); rc != DQ_OK) return -rc;
  return plan_mass(cache, s, q).bytes;
}

int dq_attention_mass(const dq_kv_cache* cache, const dq_sequences* s, const dq_heads* q, const float* lse, float scale,
                      float decay, float* mass, int64_t seq_stride, int64_t head_stride, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  if (int rc = check_mass_call(cache, s, q, true); rc != DQ_OK) return rc;
  if (int rc = check_scale(scale); rc != DQ_OK) return rc;
  if (!(decay >= 0 && decay <= 1)) return bad("decay must be in 0..1");
  if (int rc = check_mass(mass, s, cache->kv_heads, seq_stride, head_stride); rc != DQ_OK) return rc;
  if (s->batch == 0 || s->max_len == 0) return DQ_OK;
  if (int rc = check_sequence_data(s, cache); rc != DQ_OK) return rc;
  if (int rc = check_read(cache, false); rc != DQ_OK) return rc;
  if (s->tokens > 0) {
    if (int rc = check_data("q", q); rc != DQ_OK) return rc;
    if (lse == nullptr) return bad("lse: null argument");
  }
  const MassPlan p = plan_mass(cache, s, q);
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes); rc != DQ_OK) return rc;
  MassArgs m;
  m.lse = lse;
  m.decay = decay;
  m.mass = mass;
  m.seq = seq_stride;
  m.head = head_stride;
  m.splits = (int32_t)p.splits;
  if (p.splits > 1) m.part = static_cast<float*>(workspace);
  const hipError_t e = launch_attention_mass(q->dtype, cache->dtype, query_args(cache, s, q, scale), m, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "attention_mass launch");
}

int dq_kv_keep(const dq_sequences* s, int64_t kv_heads, const float* mass, int64_t seq_stride, int64_t head_stride,
               int64_t first, int64_t last, int64_t budget, int32_t* kept, int32_t* kept_lens, void* stream) {
  if (int rc = check_sequences(s, 0); rc != DQ_OK) return rc;
  if (kv_heads < 1 || kv_heads > INT32_MAX) return bad("kv_heads must be positive");
  if (s->batch >= ceil_div(kMaxGroups / 4, kv_heads)) return too_many("sequences");  // (of 1,024 threads)
  if (budget < 1 || budget > kMostKeys) return set_error(DQ_INVALID_ARGUMENT, "budget %lld", (ll)budget);
  if (first < 0 || last < 0 || first > budget || last > budget - first)
    return set_error(DQ_INVALID_ARGUMENT, "first %lld and last %lld of %lld keys", (ll)first, (ll)last, (ll)budget);
  if (int rc = check_mass(mass, s, kv_heads, seq_stride, head_stride); rc != DQ_OK) return rc;
  if (s->batch == 0) return DQ_OK;
  if (int rc = check_sequence_data(s, nullptr); rc != DQ_OK) return rc;
  if (kept == nullptr) return bad("kept: null argument");
  KeepArgs k;
  k.mass = mass;
  k.seq = seq_stride;
  k.head = head_stride;
  k.lens = s->lens;
  k.max_len = (int32_t)s->max_len;
  k.kv_heads = (int32_t)kv_heads;
  k.first = (int32_t)first;
  k.last = (int32_t)last;
  k.budget = budget;
  k.kept = kept;
  k.kept_lens = kept_lens;
  const hipError_t e = launch_kv_keep(s->batch, k, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "kv_keep launch");
}

int dq_kv_compact(const dq_kv_cache* cache, const dq_sequences* s, const int32_t* kept, int64_t budget, const int32_t* to_pages,
                  int64_t to_stride, const float* mass, float* mass_out, int64_t seq_stride, int64_t head_stride, void* stream) {
  if (int rc = check_cache(cache, false); rc != DQ_OK) return rc;
  if (int rc = check_cache_apart(cache); rc != DQ_OK) return rc;
  if (int rc = check_sequences(s, cache->page_size); rc != DQ_OK) return rc;
  if (budget < 1 || budget > kMostKeys) return set_error(DQ_INVALID_ARGUMENT, "budget %lld", (ll)budget);
  const int64_t most = std::min(budget, s->max_len);
  if (to_pages != nullptr && (to_stride < ceil_div(most, cache->page_size) || to_stride > kMostKeys))
    return set_error(DQ_INVALID_ARGUMENT, "to_stride %lld: %lld keys need %lld pages", (ll)to_stride, (ll)most,
                     (ll)ceil_div(most, cache->page_size));
  if ((mass == nullptr) != (mass_out == nullptr)) return bad("mass and mass_out go together");
  if (mass != nullptr)
    for (const float* m : {mass, static_cast<const float*>(mass_out)})
      if (int rc = check_mass(m, s, cache->kv_heads, seq_stride, head_stride); rc != DQ_OK) return rc;
  if (s->batch == 0 || s->max_len == 0) return DQ_OK;
  if (int rc = check_sequence_data(s, cache); rc != DQ_OK) return rc;
  if (int rc = check_read(cache, true); rc != DQ_OK) return rc;
  if (kept == nullptr) return bad("kept: null argument");
  // (a workgroup moves 64 rows at least)
  if (s->batch * (2 * (to_pages == nullptr ? 1 : ceil_div(most, 64)) + 1) >= kMaxGroups / cache->kv_heads) return too_many("keys");
  CompactArgs c;
  c.kept = kept;
  c.budget = budget;
  c.to_pages = to_pages;
  c.to_stride = to_stride;
  c.mass = mass;
  c.mass_out = mass_out;
  c.seq = seq_stride;
  c.head = head_stride;
  const hipError_t e = launch_kv_compact(sequence_args(cache, s), c, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "kv_compact launch");
}

}  // extern "C"
