// dq_attn.h -- the attention block's launch arguments, shared by its host checks
// (dq_attn_api.cpp) and its kernels (dq_heads.hip, dq_attn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dynaq.h"

namespace dq {

// One side of a head-rows launch: heads of `in` normalized with weight (nullptr: no norm)
// into `out`.
struct HeadRows {
  const void* in = nullptr;
  void* out = nullptr;
  const float* weight = nullptr;
  int32_t heads = 0;
  int64_t in_token = 0, in_head = 0;    // strides in values
  int64_t out_token = 0, out_head = 0;
};

struct RopeArgs {
  const float* cos = nullptr;
  const float* sin = nullptr;
  const int32_t* positions = nullptr;
  int64_t max_pos = 0;
  int32_t half = 0;  // rotated pairs of a head (0: no rotation)
  int32_t pairs = 0; // DQ_ROPE_PAIRS
};

// A cache's places: key (value) of place i of page p and head h at p * page + i * token + h * head.
struct CacheArgs {
  uint16_t* k = nullptr;
  uint16_t* v = nullptr;
  int64_t n_pages = 0;
  int64_t page = 0, token = 0, head = 0;  // strides in values
  int32_t page_size = 0;
  int32_t kv_heads = 0;
};

// Normalized and rotated head rows, two sides (q and k) in one launch. in_type / out_type: dq_float.
hipError_t launch_norm_rope(int in_type, int out_type, int64_t tokens, int dim, const HeadRows& a, const HeadRows& b,
                            float eps, const RopeArgs& rope, hipStream_t s);
// k (normalized, rotated) and v into the cache's slots; k.out and v.out are not used.
hipError_t launch_kv_append(int in_type, int cache_type, int64_t tokens, int dim, const HeadRows& k, const HeadRows& v,
                            const CacheArgs& cache, const int64_t* slots, float eps, const RopeArgs& rope,
                            hipStream_t s);

struct AttnArgs {
  CacheArgs cache;
  const void* q = nullptr;
  void* out = nullptr;
  float* lse = nullptr;
  int64_t q_token = 0, q_head = 0, out_token = 0, out_head = 0;  // strides in values
  int32_t heads = 0;  // query heads
  int32_t group = 0;  // query heads a kv head
  int32_t dim = 0;
  int32_t tokens = 0;
  int32_t batch = 0;
  int32_t max_q = 0;
  int32_t part_tokens = 0;  // tokens of this launch's sequences (at most)
  bool sliced = false;      // not the call's first sequences, or not all: their rows begin at q_offsets[0]
  const int32_t* q_offsets = nullptr;  // nullptr: one token a sequence
  const int32_t* prefix_pages = nullptr;
  const int32_t* pages = nullptr;
  const int32_t* lens = nullptr;
  int64_t pages_stride = 0;
  int32_t prefix_len = 0;
  int32_t max_len = 0;
  float scale_log2 = 0;  // scale * log2(e): the softmax runs on powers of two
  bool q_vec = false, out_vec = false;  // rows of q (out) can be read (written) in 16 (16 or 8) bytes
  float* part_o = nullptr;   // [slot][kv head][row][dim] (nullptr: one item a row, which finishes it)
  float* part_ml = nullptr;  // [slot][kv head][row] maximum (in powers of two), sum
};

// One kind of work items: (key range, kv head, row tile), for every sequence of `own` items.
struct AttnPart {
  int32_t rows = 0;    // rows of a tile: 16, 64, 128
  int32_t tiles = 0;   // row tiles (of a sequence)
  int32_t splits = 0;  // key ranges (0: no such items)
  int32_t chunk = 0;   // keys of a range, a multiple of 128
  int32_t slot = 0;    // the first range's slot of the workspace
  int32_t own_from = 0;  // with the prefix before them: where the own keys begin in the ranges
  bool with_prefix = false;
  bool backward = false;  // the last rows, which see most keys, first
};

// How a call's work is split: launches of `batch` sequences, one after another; `shared` items take the prefix with the rows of all sequences,
// `own` ones a sequence's own keys (with the prefix before them where there are no shared items).
struct AttnPlan {
  int64_t batch = 0;
  AttnPart shared, own;
  int64_t slots = 0;  // parts of a row (0: none, every item finishes its rows)
};

hipError_t launch_attention(int type, int cache_type, const AttnArgs& a, const AttnPlan& p, hipStream_t s);

}  // namespace dq
