// dq_attn_checks.h -- argument checks that the attention block's entry points share.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/dynaq.h"
#include "dq_attn.h"
#include "dq_internal.h"

namespace dq {
namespace {

typedef long long ll;

int bad(const char* what) { return set_error(DQ_INVALID_ARGUMENT, "%s", what); }

int hip_fail(hipError_t e, const char* what) {
  return set_error(e == hipErrorOutOfMemory ? DQ_OUT_OF_MEMORY : DQ_INTERNAL, "%s: %s", what, hipGetErrorString(e));
}

bool float_ok(int t) { return t == DQ_F32 || t == DQ_F16 || t == DQ_BF16; }
size_t float_bytes(int t) { return t == DQ_F32 ? 4 : 2; }

int check_dim(int64_t dim) {
  if (dim <= 0 || dim % 8 != 0) return set_error(DQ_INVALID_ARGUMENT, "head_dim %lld is not a multiple of 8", (ll)dim);
  if (dim > DQ_MAX_HEAD_DIM) return set_error(DQ_UNSUPPORTED, "head_dim %lld is over %d", (ll)dim, DQ_MAX_HEAD_DIM);
  return DQ_OK;
}

// What can be said of rows without their data: `need` heads (0: any), values addressable by int64.
int check_rows(const char* name, const dq_heads* r, int64_t tokens) {
  if (r == nullptr) return set_error(DQ_INVALID_ARGUMENT, "%s: null argument", name);
  if (!float_ok(r->dtype)) return set_error(DQ_UNSUPPORTED, "%s: type %d is not supported", name, r->dtype);
  if (r->heads <= 0) return set_error(DQ_INVALID_ARGUMENT, "%s: heads must be positive", name);
  if (r->token_stride < 0 || r->head_stride < 0) return set_error(DQ_INVALID_ARGUMENT, "%s: negative stride", name);
  const int64_t most = (int64_t)1 << 58;
  if ((tokens > 1 && r->token_stride > most / tokens) || (r->heads > 1 && r->head_stride > most / r->heads))
    return set_error(DQ_INVALID_ARGUMENT, "%s: strides too large", name);
  return DQ_OK;
}

int check_data(const char* name, const dq_heads* r) {
  if (r->p == nullptr) return set_error(DQ_INVALID_ARGUMENT, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(r->p) % float_bytes(r->dtype) != 0)
    return set_error(DQ_INVALID_ARGUMENT, "%s: misaligned pointer", name);
  return DQ_OK;
}

// An output's rows must not run into each other.
int check_apart(const char* name, const dq_heads* r, int64_t tokens, int64_t dim) {
  const int64_t th = r->head_stride, tt = r->token_stride, nh = r->heads;
  if (nh > 1 && th < dim) return set_error(DQ_INVALID_ARGUMENT, "%s: head_stride %lld < head_dim %lld", name, (ll)th, (ll)dim);
  if (tokens > 1 && tt < dim)
    return set_error(DQ_INVALID_ARGUMENT, "%s: token_stride %lld < head_dim %lld", name, (ll)tt, (ll)dim);
  if (tokens > 1 && nh > 1 && tt < (nh - 1) * th + dim && th < (tokens - 1) * tt + dim)
    return set_error(DQ_INVALID_ARGUMENT, "%s: tokens and heads overlap (strides %lld, %lld)", name, (ll)tt, (ll)th);
  return DQ_OK;
}

int check_cache(const dq_kv_cache* c, bool data) {
  if (c == nullptr) return bad("cache: null argument");
  if (c->dtype != DQ_F16 && c->dtype != DQ_BF16) return set_error(DQ_UNSUPPORTED, "cache: type %d is not supported", c->dtype);
  if (int rc = check_dim(c->head_dim); rc != DQ_OK) return rc;
  if (c->kv_heads <= 0) return bad("cache: kv_heads must be positive");
  if (c->page_size <= 0 || c->page_size % 16 != 0)
    return set_error(DQ_INVALID_ARGUMENT, "cache: page_size %d is not a multiple of 16", c->page_size);
  if (c->n_pages < 0 || c->n_pages > INT32_MAX) return set_error(DQ_INVALID_ARGUMENT, "cache: n_pages %lld", (ll)c->n_pages);
  for (int64_t st : {c->page_stride, c->token_stride, c->head_stride})
    if (st < 0 || st % 8 != 0 || st > ((int64_t)1 << 58) / (st == c->page_stride ? c->n_pages + 1 : c->page_size + c->kv_heads))
      return set_error(DQ_INVALID_ARGUMENT, "cache: stride %lld is negative, no multiple of 8 or too large", (ll)st);
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
      return set_error(DQ_INVALID_ARGUMENT, "cache: places overlap (page_stride %lld, token_stride %lld, head_stride %lld)",
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

CacheArgs cache_args(const dq_kv_cache* c) {
  return CacheArgs{static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->n_pages, c->page_stride,
                       c->token_stride, c->head_stride, c->page_size, c->kv_heads};
}

constexpr float kLog2e = 1.44269504088896340736f;
// Workgroups of an attention launch stay below this: a dispatch counts its threads, 256 a workgroup, in 32 bits.
constexpr int64_t kMaxGroups = (int64_t)1 << 24;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned(const dq_heads* r, size_t bytes) {
  const size_t v = float_bytes(r->dtype);
  return reinterpret_cast<uintptr_t>(r->p) % bytes == 0 && r->token_stride * v % bytes == 0 && r->head_stride * v % bytes == 0;
}

}  // namespace
}  // namespace dq
