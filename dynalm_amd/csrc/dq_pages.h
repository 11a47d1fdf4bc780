// dq_pages.h -- launch arguments of the long caches' operators, shared by their host checks
// (dq_pages_api.cpp) and their kernels (dq_pages.hip, dq_evict.hip). The sequences, rows and pages
// of a call are those of AttnArgs (prefix_len 0).
#pragma once

#include <type_traits>

#include "dq_attn.h"

namespace dq {

// Bounds of the pages of keys [from[b], lens[b]): `slots` pages of a sequence at most.
hipError_t launch_page_bounds(int cache_type, const AttnArgs& a, const int32_t* from, int64_t slots, uint16_t* bounds,
                              hipStream_t s);

struct ChooseArgs {
  const uint16_t* bounds = nullptr;
  int32_t* chosen = nullptr;
  uint64_t* keys = nullptr;  // [token of the launch][kv head][page]: the interval of a score (two floats), or the 64-bit score in an order of whole numbers
  int32_t pages = 0;         // of a sequence, at most
  int32_t first = 0, last = 0;
  int64_t count = 0;
  int64_t tokens = 0;        // of a launch
};
hipError_t launch_choose_pages(int type, int cache_type, const AttnArgs& a, const ChooseArgs& c, hipStream_t s);

// `splits` ranges of `chunk` entries of a row's list each; with a.part_o their parts are joined.
hipError_t launch_page_attention(int type, int cache_type, const AttnArgs& a, const int32_t* chosen, int64_t count,
                                 int32_t splits, int32_t chunk, hipStream_t s);

struct MassArgs {
  const float* lse = nullptr;
  float decay = 0;
  float* mass = nullptr;
  int64_t seq = 0, head = 0;  // strides in values
  float* part = nullptr;      // [part][sequence][kv head][key] (nullptr: one part, added at once)
  int32_t splits = 1;         // parts of a sequence's rows
};
hipError_t launch_attention_mass(int type, int cache_type, const AttnArgs& a, const MassArgs& m, hipStream_t s);

struct KeepArgs {
  const float* mass = nullptr;
  int64_t seq = 0, head = 0;  // strides in values
  const int32_t* lens = nullptr;
  int32_t max_len = 0;
  int32_t kv_heads = 0;
  int32_t first = 0, last = 0;
  int64_t budget = 0;
  int32_t* kept = nullptr;
  int32_t* kept_lens = nullptr;
};
hipError_t launch_kv_keep(int64_t batch, const KeepArgs& k, hipStream_t s);

struct CompactArgs {
  const int32_t* kept = nullptr;
  int64_t budget = 0;
  const int32_t* to_pages = nullptr;  // nullptr: in place
  int64_t to_stride = 0;
  const float* mass = nullptr;
  float* mass_out = nullptr;
  int64_t seq = 0, head = 0;  // strides in values
};
hipError_t launch_kv_compact(const AttnArgs& a, const CompactArgs& c, hipStream_t s);

// The join of dq_attn.hip: rows' parts [range][kv head][row] of `splits` ranges.
hipError_t launch_join(int type, int cache_type, const AttnArgs& a, int32_t splits, hipStream_t s);

// f(query type, cache type), as constants.
template <class F>
inline hipError_t by_types(int type, int cache_type, F&& f) {
  using f32 = std::integral_constant<int, DQ_F32>;
  using f16 = std::integral_constant<int, DQ_F16>;
  using bf16 = std::integral_constant<int, DQ_BF16>;
  if (cache_type == DQ_F16) return type == DQ_F32 ? f(f32{}, f16{}) : f(f16{}, f16{});
  return type == DQ_F32 ? f(f32{}, bf16{}) : f(bf16{}, bf16{});
}

}  // namespace dq
