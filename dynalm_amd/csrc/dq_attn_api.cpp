// dq_attn_api.cpp -- the attention block's C ABI (declared in include/dynaq.h): argument
// checks with dynacore's status codes, then the launches. Nothing is allocated or kept.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/dynaq.h"
#include "dq_attn.h"
#include "dq_internal.h"

namespace {

typedef long long ll;

int bad(const char* what) { return dq::set_error(DQ_INVALID_ARGUMENT, "%s", what); }

int hip_fail(hipError_t e, const char* what) {
  return dq::set_error(e == hipErrorOutOfMemory ? DQ_OUT_OF_MEMORY : DQ_INTERNAL, "%s: %s", what, hipGetErrorString(e));
}

bool float_ok(int t) { return t == DQ_F32 || t == DQ_F16 || t == DQ_BF16; }
size_t float_bytes(int t) { return t == DQ_F32 ? 4 : 2; }

int check_dim(int64_t dim) {
  if (dim <= 0 || dim % 8 != 0) return dq::set_error(DQ_INVALID_ARGUMENT, "head_dim %lld is not a multiple of 8", (ll)dim);
  if (dim > DQ_MAX_HEAD_DIM) return dq::set_error(DQ_UNSUPPORTED, "head_dim %lld is over %d", (ll)dim, DQ_MAX_HEAD_DIM);
  return DQ_OK;
}

// What can be said of rows without their data: `need` heads (0: any), values addressable by int64.
int check_rows(const char* name, const dq_heads* r, int64_t tokens) {
  if (r == nullptr) return dq::set_error(DQ_INVALID_ARGUMENT, "%s: null argument", name);
  if (!float_ok(r->dtype)) return dq::set_error(DQ_UNSUPPORTED, "%s: type %d is not supported", name, r->dtype);
  if (r->heads <= 0) return dq::set_error(DQ_INVALID_ARGUMENT, "%s: heads must be positive", name);
  if (r->token_stride < 0 || r->head_stride < 0) return dq::set_error(DQ_INVALID_ARGUMENT, "%s: negative stride", name);
  const int64_t most = (int64_t)1 << 58;
  if ((tokens > 1 && r->token_stride > most / tokens) || (r->heads > 1 && r->head_stride > most / r->heads))
    return dq::set_error(DQ_INVALID_ARGUMENT, "%s: strides too large", name);
  return DQ_OK;
}

int check_data(const char* name, const dq_heads* r) {
  if (r->p == nullptr) return dq::set_error(DQ_INVALID_ARGUMENT, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(r->p) % float_bytes(r->dtype) != 0)
    return dq::set_error(DQ_INVALID_ARGUMENT, "%s: misaligned pointer", name);
  return DQ_OK;
}

// An output's rows must not run into each other.
int check_apart(const char* name, const dq_heads* r, int64_t tokens, int64_t dim) {
  const int64_t th = r->head_stride, tt = r->token_stride, nh = r->heads;
  if (nh > 1 && th < dim) return dq::set_error(DQ_INVALID_ARGUMENT, "%s: head_stride %lld < head_dim %lld", name, (ll)th, (ll)dim);
  if (tokens > 1 && tt < dim)
    return dq::set_error(DQ_INVALID_ARGUMENT, "%s: token_stride %lld < head_dim %lld", name, (ll)tt, (ll)dim);
  if (tokens > 1 && nh > 1 && tt < (nh - 1) * th + dim && th < (tokens - 1) * tt + dim)
    return dq::set_error(DQ_INVALID_ARGUMENT, "%s: tokens and heads overlap (strides %lld, %lld)", name, (ll)tt, (ll)th);
  return DQ_OK;
}

int check_rope(const dq_rope* r, const int32_t* positions, int64_t dim, int64_t tokens, dq::RopeArgs* out) {
  if (r == nullptr) return DQ_OK;
  if (r->style != DQ_ROPE_HALVES && r->style != DQ_ROPE_PAIRS)
    return dq::set_error(DQ_INVALID_ARGUMENT, "unknown rotation style %d", r->style);
  if (r->rot_dim < 2 || r->rot_dim % 2 != 0 || r->rot_dim > dim)
    return dq::set_error(DQ_INVALID_ARGUMENT, "rot_dim %d is not even and in 2..head_dim %lld", r->rot_dim, (ll)dim);
  if (r->max_pos < 0) return bad("max_pos must be >= 0");
  if (tokens > 0 && (positions == nullptr || ((r->cos == nullptr || r->sin == nullptr) && r->max_pos > 0)))
    return bad("rotation: null argument");
  *out = dq::RopeArgs{r->cos, r->sin, positions, r->max_pos, r->rot_dim / 2, r->style == DQ_ROPE_PAIRS};
  return DQ_OK;
}

int check_eps(const float* weight, float eps) {
  if (weight != nullptr && !(eps >= 0 && std::isfinite(eps))) return bad("eps must be finite and >= 0");
  return DQ_OK;
}

int check_cache(const dq_kv_cache* c, bool data) {
  if (c == nullptr) return bad("cache: null argument");
  if (c->dtype != DQ_F16 && c->dtype != DQ_BF16) return dq::set_error(DQ_UNSUPPORTED, "cache: type %d is not supported", c->dtype);
  if (int rc = check_dim(c->head_dim); rc != DQ_OK) return rc;
  if (c->kv_heads <= 0) return bad("cache: kv_heads must be positive");
  if (c->page_size <= 0 || c->page_size % 16 != 0)
    return dq::set_error(DQ_INVALID_ARGUMENT, "cache: page_size %d is not a multiple of 16", c->page_size);
  if (c->n_pages < 0 || c->n_pages > INT32_MAX) return dq::set_error(DQ_INVALID_ARGUMENT, "cache: n_pages %lld", (ll)c->n_pages);
  for (int64_t st : {c->page_stride, c->token_stride, c->head_stride})
    if (st < 0 || st % 8 != 0 || st > ((int64_t)1 << 58) / (st == c->page_stride ? c->n_pages + 1 : c->page_size + c->kv_heads))
      return dq::set_error(DQ_INVALID_ARGUMENT, "cache: stride %lld is negative, no multiple of 8 or too large", (ll)st);
  if (c->token_stride < c->head_dim || (c->kv_heads > 1 && c->head_stride < c->head_dim) || (c->n_pages > 1 && c->page_stride < c->head_dim))
    return bad("cache: a stride is less than head_dim");
  if (data && c->n_pages > 0) {
    if (c->k == nullptr || c->v == nullptr) return bad("cache: null pointer");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 != 0) return bad("cache: k and v must be 16-byte aligned");
  }
  return DQ_OK;
}

// A cache's places that are written must not run into each other, nor its keys into its values.
int check_cache_apart(const dq_kv_cache* c) {
  if (c->n_pages == 0) return DQ_OK;
  struct Axis {
    int64_t stride, n;
  } x[3] = {{c->page_stride, c->n_pages}, {c->token_stride, c->page_size}, {c->head_stride, c->kv_heads}};
  for (Axis& a : x)
    if (a.n == 1) a.stride = 0;
  std::sort(x, x + 3, [](const Axis& a, const Axis& b) { return a.stride < b.stride; });
  int64_t end = c->head_dim;  // of the values that the shorter strides reach
  for (const Axis& a : x) {
    if (a.n > 1 && a.stride < end)
      return dq::set_error(DQ_INVALID_ARGUMENT, "cache: places overlap (page_stride %lld, token_stride %lld, head_stride %lld)",
                           (ll)c->page_stride, (ll)c->token_stride, (ll)c->head_stride);
    end += (a.n - 1) * a.stride;
  }
  // Apart by d values, a key's place meets a value's if d is less than a head away from a difference of two places;
  // of each axis, longest stride first, only the two multiples next to d can come that near.
  const int64_t d = (reinterpret_cast<intptr_t>(c->v) - reinterpret_cast<intptr_t>(c->k)) / 2;
  for (int pick = 0; pick < 8; ++pick) {
    int64_t rest = d < 0 ? -d : d;
    for (int i = 2; i >= 0; --i) {
      if (x[i].n == 1) continue;
      int64_t m = rest / x[i].stride + (pick >> i & 1);
      if (rest < 0) m = -(-rest / x[i].stride) - (pick >> i & 1);
      m = std::min(std::max(m, -(x[i].n - 1)), x[i].n - 1);
      rest -= m * x[i].stride;
    }
    if (rest < c->head_dim && -rest < c->head_dim) return bad("cache: keys and values overlap");
  }
  return DQ_OK;
}

dq::CacheArgs cache_args(const dq_kv_cache* c) {
  return dq::CacheArgs{static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->n_pages, c->page_stride,
                       c->token_stride, c->head_stride, c->page_size, c->kv_heads};
}

dq::HeadRows rows(const dq_heads* in, const dq_heads* out, const float* w) {
  dq::HeadRows r;
  r.in = in->p;
  r.weight = w;
  r.heads = in->heads;
  r.in_token = in->token_stride;
  r.in_head = in->head_stride;
  if (out != nullptr) {
    r.out = out->p;
    r.out_token = out->token_stride;
    r.out_head = out->head_stride;
  }
  return r;
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int64_t kMaxRows = (int64_t)1 << 31;   // head rows of a call: they are counted in 32 bits
constexpr int64_t kMaxHeads = (int64_t)1 << 25;  // heads of a token: its rows run in one launch

// Workgroups of an attention launch stay below this: a dispatch counts its threads, 256 a workgroup, in 32 bits.
constexpr int64_t kMaxGroups = (int64_t)1 << 24;
// Rows of a sequence that fill tiles by themselves: from here on it reads the prefix for itself.
constexpr int64_t kFullRows = 64;

int check_tokens(int64_t tokens, int64_t heads) {
  if (tokens < 0) return bad("tokens must be >= 0");
  if (tokens > kMaxRows / heads || heads > kMaxHeads) return dq::set_error(DQ_UNSUPPORTED, "%lld tokens of %lld heads are too many", (ll)tokens, (ll)heads);
  return DQ_OK;
}

int check_attention(const dq_kv_cache* c, const dq_attention* a, bool data) {
  if (a == nullptr) return bad("null argument");
  if (int rc = check_cache(c, data); rc != DQ_OK) return rc;
  if (a->tokens < 0 || a->batch < 0) return bad("tokens and batch must be >= 0");
  if (int rc = check_rows("q", a->q, a->tokens); rc != DQ_OK) return rc;
  if (int rc = check_rows("out", a->out, a->tokens); rc != DQ_OK) return rc;
  if (int rc = check_apart("out", a->out, a->tokens, c->head_dim); rc != DQ_OK) return rc;
  if (a->q->dtype != a->out->dtype || (a->q->dtype != DQ_F32 && a->q->dtype != c->dtype))
    return dq::set_error(DQ_UNSUPPORTED, "q type %d, out type %d with cache type %d: q and out have the cache's type or fp32",
                         a->q->dtype, a->out->dtype, c->dtype);
  if (a->q->heads != a->out->heads || a->q->heads % c->kv_heads != 0)
    return dq::set_error(DQ_INVALID_ARGUMENT, "%d query heads, %d of out, %d kv heads", a->q->heads, a->out->heads, c->kv_heads);
  if (c->token_stride > (1 << 25)) return dq::set_error(DQ_UNSUPPORTED, "cache: token_stride %lld", (ll)c->token_stride);
  // Head rows and work items are counted in 32 bits.
  if (a->tokens > ((int64_t)1 << 30) / a->q->heads)
    return dq::set_error(DQ_UNSUPPORTED, "%lld tokens of %d heads are too many", (ll)a->tokens, a->q->heads);
  if (a->max_q < 1) return dq::set_error(DQ_INVALID_ARGUMENT, "max_q %lld", (ll)a->max_q);
  const int64_t most_q = a->max_q < a->tokens ? a->max_q : a->tokens;
  if (a->batch > INT32_MAX / 2 / a->q->heads || a->batch * (most_q * (a->q->heads / c->kv_heads) / 16 + 1) > INT32_MAX / 2 / c->kv_heads)
    return dq::set_error(DQ_UNSUPPORTED, "%lld sequences of up to %lld tokens are too many", (ll)a->batch, (ll)a->max_q);
  if ((most_q * (a->q->heads / c->kv_heads) / kFullRows + 1) * c->kv_heads >= kMaxGroups)  // (of one sequence)
    return dq::set_error(DQ_UNSUPPORTED, "%lld tokens of %d heads are too many for a launch", (ll)most_q, a->q->heads);
  if (data && a->q_offsets == nullptr && (a->tokens != a->batch || a->max_q != 1))
    return bad("without q_offsets every sequence has one token");
  const int64_t most = (int64_t)1 << 29;
  if (a->prefix_len < 0 || a->prefix_len > most || a->max_len < 0 || a->max_len > most)
    return dq::set_error(DQ_INVALID_ARGUMENT, "prefix_len %lld, max_len %lld: 0..2^29 keys", (ll)a->prefix_len, (ll)a->max_len);
  if (a->pages_stride < (a->max_len + c->page_size - 1) / c->page_size || a->pages_stride > most)
    return dq::set_error(DQ_INVALID_ARGUMENT, "pages_stride %lld: max_len %lld needs %lld pages", (ll)a->pages_stride, (ll)a->max_len,
                         (ll)((a->max_len + c->page_size - 1) / c->page_size));
  if (!(a->scale > 0) || !std::isfinite(a->scale * kLog2e)) return bad("scale must be positive and finite");
  return DQ_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Items a launch aims at: two run on each of the 256 CUs at once. Shared ones take the rows of the whole
// batch and compute for long, own ones beside them read: one shared item for each CU. 64 sequences, 32 / 8
// bf16 heads of 128, 8,192 shared and up to 512 own keys: 128 shared items 54.3 us, 256 44.0, 384 47.6, 512
// 49.8; 128 sequences, 32 / 4 heads, 32,768 and up to 2,048 keys: 214, 141, 139, 140. Own items of 512
// against 1,024 on the same: 52.4 and 55.1, 140 and 151 (more ranges are more parts to write and to join).
constexpr int64_t kSharedItems = 256, kOwnItems = 512;
// Keys that are worth an item of their own (128: 20.2 us against 19.3 on 32 short sequences, 15.9 against
// 16.4 on 7).
constexpr int64_t kLeastKeys = 256;

// Keys of a prefix from which on a batch too large for the workspace runs in slices that share it. 4,100 / 8,192 sequences, 32 / 8
// bf16 heads of 128, slices against every sequence's own reading: 128 keys 429 / 964 against 306 / 744 us, 256 keys 439 /
// 981 against 403 / 941, 512 keys 448 / 992 against 652 / 1,460, 1,024 keys 473 / 1,044 against 1,212 / 2,599.
constexpr int64_t kSliceKeys = 288;

// Rows times keys (of all kv heads) up to which shared items take 64 rows and not 128: more items, each
// sooner done. 105 / 128 / 192 / 256 rows on 1,111 / 8,192 / 8,192 / 8,192 keys of 5 / 8 / 8 / 8 heads: 14.1
// against 16.4, 29.3 against 35.4, 38.0 against 39.1, 43.8 against 46.5 us; 128 rows on 32,768 keys of 8: 57.0 and 53.6.
constexpr int64_t kSmallShared = 24 << 20;

// Ranges of `keys` keys for `items` row tiles: as many as bring the items to `target`, of kLeastKeys keys at least.
void split_keys(dq::AttnPart* p, int64_t items, int64_t keys, int64_t target) {
  int64_t n = target / items;
  n = n < ceil_div(keys, kLeastKeys) ? n : ceil_div(keys, kLeastKeys);
  n = n > 1 ? n : 1;
  p->chunk = (int32_t)(ceil_div(ceil_div(keys, n), 128) * 128);
  if (p->chunk == 0) p->chunk = 128;
  p->splits = (int32_t)(keys > 0 ? ceil_div(keys, p->chunk) : 1);
}

// The most tokens that a sequence, that `batch` of them can have.
int64_t most_tokens(const dq_attention* a, int64_t batch) {
  const int64_t max_q = std::min(a->max_q, a->tokens);
  return max_q > a->tokens / batch ? a->tokens : std::min(a->tokens, batch * max_q);
}

// Bytes of the parts: O and (m, l) of every slot.
int64_t part_bytes(const dq_kv_cache* c, const dq_attention* a, int64_t tokens, int64_t slots) {
  return slots * tokens * a->q->heads * (c->head_dim + 2) * 4;
}

// The plan of a launch of `batch` sequences.
dq::AttnPlan plan_launch(const dq_kv_cache* c, const dq_attention* a, int64_t batch) {
  const int64_t group = a->q->heads / c->kv_heads, tokens = most_tokens(a, batch), all = tokens * group;
  const int64_t rows = std::min(a->max_q, a->tokens) * group;
  const bool f32 = a->q->dtype == DQ_F32;
  // (128 rows of fp32 or of heads over 128 values would leave one wave a SIMD: 864 GFLOP of prompts behind a prefix in
  // heads of 256, 1,143 to 1,174 us with 64 rows against 1,776)
  const bool wide = !f32 && c->head_dim <= 128;
  auto tile = [&](int64_t n) { return n <= 16 ? 16 : n <= 64 || !wide ? 64 : 128; };
  dq::AttnPlan p;
  for (int less = 0;; ++less) {  // (fewer parts where they would not fit the workspace; at last none)
    p = dq::AttnPlan{};
    p.batch = batch;
    p.own.rows = tile(rows);
    p.own.tiles = (int32_t)ceil_div(rows, p.own.rows);
    p.own.backward = true;
    // The prefix with all sequences' rows, unless one sequence's rows fill tiles by themselves.
    if (a->prefix_len > 0 && batch > 1 && rows < kFullRows && (kSharedItems >> less) > 0) {
      p.shared.rows = all > 16 && all * a->prefix_len * c->kv_heads <= kSmallShared ? 64 : tile(all);
      p.shared.tiles = (int32_t)ceil_div(all, p.shared.rows);
      split_keys(&p.shared, p.shared.tiles * c->kv_heads, a->prefix_len, kSharedItems >> less);
      if (a->max_len > 0) {
        split_keys(&p.own, batch * p.own.tiles * c->kv_heads, a->max_len, kOwnItems >> less);
        p.own.slot = p.shared.splits;
      }
    } else {
      p.own.with_prefix = a->prefix_len > 0;
      p.own.own_from = (int32_t)(ceil_div(a->prefix_len, 128) * 128);
      const int64_t items = batch * p.own.tiles * c->kv_heads;
      split_keys(&p.own, items, p.own.own_from + a->max_len, kOwnItems >> less);
    }
    const int64_t slots = p.shared.splits + p.own.splits;
    p.slots = slots > 1 ? slots : 0;
    if (part_bytes(c, a, tokens, p.slots) <= (int64_t)DQ_ATTENTION_WORKSPACE_BYTES) return p;
  }
}

int64_t workgroups(const dq_kv_cache* c, const dq::AttnPlan& p) {
  return ((int64_t)p.shared.tiles * p.shared.splits + (int64_t)p.own.tiles * p.own.splits * p.batch) * c->kv_heads;
}

// A batch of more items than a launch takes runs in slices of whole sequences, and so does one whose rows leave more than the
// workspace in two parts each (a shared one and an own one), so that the prefix is read once a slice and not once a
// sequence; a prefix of less than kSliceKeys keys is read by every sequence then.
dq::AttnPlan plan(const dq_kv_cache* c, const dq_attention* a) {
  int64_t batch = a->batch;
  const int64_t max_q = std::min(a->max_q, a->tokens);
  if (a->prefix_len >= kSliceKeys && a->max_len > 0 && batch > 1 && max_q * (a->q->heads / c->kv_heads) < kFullRows) {
    const int64_t fit = (int64_t)DQ_ATTENTION_WORKSPACE_BYTES / part_bytes(c, a, 1, 2);
    if (a->tokens > fit && fit >= 2 * max_q) batch = ceil_div(batch, ceil_div(batch, fit / max_q));
  }
  dq::AttnPlan p = plan_launch(c, a, batch);
  while (batch > 1 && workgroups(c, p) >= kMaxGroups) p = plan_launch(c, a, batch = ceil_div(batch, 2));
  return p;
}

// The launch of `batch` sequences from sequence b on, of a call in launches of p.batch.
hipError_t launch_slice(const dq_kv_cache* c, const dq_attention* a, const dq::AttnPlan& p, dq::AttnArgs r, int64_t b, hipStream_t s) {
  const int64_t batch = std::min(p.batch, a->batch - b);
  r.batch = (int32_t)batch;
  r.part_tokens = (int32_t)most_tokens(a, batch);
  r.lens = a->max_len > 0 ? a->lens + b : nullptr;
  r.pages = a->max_len > 0 ? a->pages + b * a->pages_stride : nullptr;
  if (a->q_offsets != nullptr) {
    r.q_offsets = a->q_offsets + b;
    r.tokens = (int32_t)a->tokens;
    r.sliced = batch < a->batch;
  } else {  // one token each
    const int64_t bytes = float_bytes(a->q->dtype);
    r.tokens = (int32_t)batch;
    r.q = static_cast<const char*>(r.q) + b * r.q_token * bytes;
    r.out = static_cast<char*>(r.out) + b * r.out_token * bytes;
    if (r.lse != nullptr) r.lse += b * r.heads;
  }
  return dq::launch_attention(a->q->dtype, c->dtype, r, p, s);
}

bool aligned(const dq_heads* r, size_t bytes) {
  const size_t v = float_bytes(r->dtype);
  return reinterpret_cast<uintptr_t>(r->p) % bytes == 0 && r->token_stride * v % bytes == 0 && r->head_stride * v % bytes == 0;
}

dq::AttnArgs attn_args(const dq_kv_cache* c, const dq_attention* a) {
  dq::AttnArgs r;
  r.cache = cache_args(c);
  r.q = a->q->p;
  r.out = a->out->p;
  r.lse = a->lse;
  r.q_token = a->q->token_stride;
  r.q_head = a->q->head_stride;
  r.out_token = a->out->token_stride;
  r.out_head = a->out->head_stride;
  r.heads = a->q->heads;
  r.group = a->q->heads / c->kv_heads;
  r.dim = c->head_dim;
  r.max_q = (int32_t)std::min(a->max_q, a->tokens);
  r.prefix_pages = a->prefix_pages;
  r.pages_stride = a->pages_stride;
  r.prefix_len = (int32_t)a->prefix_len;
  r.max_len = (int32_t)a->max_len;
  r.scale_log2 = std::fmax(a->scale * kLog2e, 1.2e-38f);
  r.q_vec = aligned(a->q, 16);
  r.out_vec = aligned(a->out, 4 * float_bytes(a->out->dtype));
  return r;
}

}  // namespace

extern "C" {

int dq_qk_norm_rope(int64_t tokens, int64_t head_dim, const dq_heads* q, const dq_heads* q_out, const float* q_weight,
                    const dq_heads* k, const dq_heads* k_out, const float* k_weight, float eps, const dq_rope* rope,
                    const int32_t* positions, void* stream) {
  if (int rc = check_dim(head_dim); rc != DQ_OK) return rc;
  if ((k == nullptr) != (k_out == nullptr)) return bad("k and k_out go together");
  const int sides = k != nullptr ? 2 : 1;
  const dq_heads* const in[2] = {q, k};
  const dq_heads* const out[2] = {q_out, k_out};
  const char* const in_name[2] = {"q", "k"};
  const char* const out_name[2] = {"q_out", "k_out"};
  int64_t heads = 0;
  for (int i = 0; i < sides; ++i) {
    if (int rc = check_rows(in_name[i], in[i], tokens); rc != DQ_OK) return rc;
    if (int rc = check_rows(out_name[i], out[i], tokens); rc != DQ_OK) return rc;
    if (int rc = check_apart(out_name[i], out[i], tokens, head_dim); rc != DQ_OK) return rc;
    if (in[i]->heads != out[i]->heads)
      return dq::set_error(DQ_INVALID_ARGUMENT, "%s: %d heads into %d", in_name[i], in[i]->heads, out[i]->heads);
    if (in[i]->dtype != q->dtype || out[i]->dtype != q_out->dtype)
      return dq::set_error(DQ_UNSUPPORTED, "q and k differ in type");
    heads += in[i]->heads;
  }
  if (int rc = check_tokens(tokens, heads); rc != DQ_OK) return rc;
  if (int rc = check_eps(q_weight != nullptr ? q_weight : k_weight, eps); rc != DQ_OK) return rc;
  dq::RopeArgs ra;
  if (int rc = check_rope(rope, positions, head_dim, tokens, &ra); rc != DQ_OK) return rc;
  if (tokens == 0) return DQ_OK;
  for (int i = 0; i < sides; ++i) {
    if (int rc = check_data(in_name[i], in[i]); rc != DQ_OK) return rc;
    if (int rc = check_data(out_name[i], out[i]); rc != DQ_OK) return rc;
  }
  dq::HeadRows a = rows(q, q_out, q_weight), b;
  if (k != nullptr) b = rows(k, k_out, k_weight);
  const hipError_t e = dq::launch_norm_rope(q->dtype, q_out->dtype, tokens, (int)head_dim, a, b, eps, ra, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "qk_norm_rope launch");
}

int dq_kv_append(const dq_kv_cache* cache, int64_t tokens, const dq_heads* k, const dq_heads* v, const int64_t* slots,
                 const float* k_weight, float eps, const dq_rope* rope, const int32_t* positions, void* stream) {
  if (int rc = check_cache(cache, tokens > 0); rc != DQ_OK) return rc;
  if (int rc = check_rows("k", k, tokens); rc != DQ_OK) return rc;
  if (int rc = check_rows("v", v, tokens); rc != DQ_OK) return rc;
  if (k->dtype != v->dtype) return dq::set_error(DQ_UNSUPPORTED, "k and v differ in type");
  if (k->heads != cache->kv_heads || v->heads != cache->kv_heads)
    return dq::set_error(DQ_INVALID_ARGUMENT, "%d and %d heads, the cache has %d", k->heads, v->heads, cache->kv_heads);
  if (int rc = check_tokens(tokens, 2 * (int64_t)cache->kv_heads); rc != DQ_OK) return rc;
  if (int rc = check_eps(k_weight, eps); rc != DQ_OK) return rc;
  dq::RopeArgs ra;
  if (int rc = check_rope(rope, positions, cache->head_dim, tokens, &ra); rc != DQ_OK) return rc;
  if (tokens == 0) return DQ_OK;
  if (int rc = check_cache_apart(cache); rc != DQ_OK) return rc;
  if (slots == nullptr) return bad("slots: null argument");
  if (int rc = check_data("k", k); rc != DQ_OK) return rc;
  if (int rc = check_data("v", v); rc != DQ_OK) return rc;
  if (cache->n_pages == 0) return DQ_OK;  // no slot is inside
  const hipError_t e = dq::launch_kv_append(k->dtype, cache->dtype, tokens, cache->head_dim, rows(k, nullptr, k_weight),
                                            rows(v, nullptr, nullptr), cache_args(cache), slots, eps, ra,
                                            static_cast<hipStream_t>(stream));
  return e == hipSuccess ? DQ_OK : hip_fail(e, "kv_append launch");
}

int64_t dq_shared_attention_workspace(const dq_kv_cache* cache, const dq_attention* a) {
  if (int rc = check_attention(cache, a, false); rc != DQ_OK) return -rc;
  if (a->tokens == 0 || a->batch == 0) return 0;
  const dq::AttnPlan p = plan(cache, a);
  return part_bytes(cache, a, most_tokens(a, p.batch), p.slots);
}

int dq_shared_attention(const dq_kv_cache* cache, const dq_attention* a, void* workspace, int64_t workspace_bytes,
                        void* stream) {
  if (int rc = check_attention(cache, a, true); rc != DQ_OK) return rc;
  if (a->tokens == 0 || a->batch == 0) return DQ_OK;
  if (int rc = check_data("q", a->q); rc != DQ_OK) return rc;
  if (int rc = check_data("out", a->out); rc != DQ_OK) return rc;
  if (a->prefix_len > 0 && a->prefix_pages == nullptr) return bad("prefix_pages: null argument");
  if (a->max_len > 0 && (a->pages == nullptr || a->lens == nullptr)) return bad("pages, lens: null argument");
  if (cache->n_pages == 0 && (a->prefix_len > 0 || a->max_len > 0)) return bad("cache: no pages");
  const dq::AttnPlan p = plan(cache, a);
  dq::AttnArgs args = attn_args(cache, a);
  if (p.slots > 0) {
    const int64_t tokens = most_tokens(a, p.batch), need = part_bytes(cache, a, tokens, p.slots);
    if (workspace == nullptr) return bad("workspace: null argument");
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return bad("workspace: must be 16-byte aligned");
    if (workspace_bytes < need)
      return dq::set_error(DQ_RESOURCE_EXHAUSTED, "workspace: %lld bytes, the call needs %lld", (ll)workspace_bytes, (ll)need);
    args.part_o = static_cast<float*>(workspace);
    args.part_ml = args.part_o + p.slots * tokens * a->q->heads * cache->head_dim;
  }
  for (int64_t b = 0; b < a->batch; b += p.batch)
    if (const hipError_t e = launch_slice(cache, a, p, args, b, static_cast<hipStream_t>(stream)); e != hipSuccess)
      return hip_fail(e, "shared_attention launch");
  return DQ_OK;
}

}  // extern "C"
