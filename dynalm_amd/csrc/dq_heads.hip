// dq_heads.hip -- norms and rotation of query and key heads, and the append of keys and
// values to a paged cache with both on the way.
//
// A head row is D <= 256 values: y = x / sqrt(mean x^2 + eps) * w, then the first 2 * half of
// them turn in pairs, a' = a c - b s, b' = b c + a s. One wave a row: every value is read once
// and written once.
#include <type_traits>

#include "dq_attn.h"
#include "dq_device.h"

namespace dq {
namespace {

template <int T>
DQ_DEV float load1(const void* p, int64_t i) {
  if constexpr (T == DQ_F32) return static_cast<const float*>(p)[i];
  const u32 h = static_cast<const uint16_t*>(p)[i];
  if constexpr (T == DQ_F16) return h2f(h);
  return as_f(h << 16);
}

template <int T>
DQ_DEV void store1(void* p, int64_t i, float x) {
  if constexpr (T == DQ_F32)
    static_cast<float*>(p)[i] = x;
  else if constexpr (T == DQ_F16)
    static_cast<uint16_t*>(p)[i] = f2h(x);
  else
    static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, (__bf16)x);
}

DQ_DEV float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// A wave's head row: value lane + 64 j of it at out[j], after norm and rotation. The pair's other
// value is read again (the line is in the cache), so no lane needs another's.
template <int T>
DQ_DEV void head_row(const void* x, int64_t base, int dim, const float* w, float eps, const RopeArgs& rp, int64_t t,
                     int lane, float (&out)[4]) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = lane + 64 * j < dim ? load1<T>(x, base + lane + 64 * j) : 0.f;
  float r = 1.f;
  if (w != nullptr) {
    float s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) s += v[j] * v[j];
    r = 1.f / sqrtf(wave_sum(s) / (float)dim + eps);
  }
  const int64_t pos = rp.half > 0 ? rp.positions[t] : 0;
  const bool inside = pos >= 0 && pos < rp.max_pos;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = lane + 64 * j;
    if (d >= dim) continue;
    float y = w != nullptr ? v[j] * r * w[d] : v[j];
    if (d < 2 * rp.half) {
      const int pair = rp.pairs ? d >> 1 : d < rp.half ? d : d - rp.half;
      const bool first = rp.pairs ? (d & 1) == 0 : d < rp.half;
      const int o = rp.pairs ? d ^ 1 : first ? d + rp.half : d - rp.half;
      float z = load1<T>(x, base + o);
      if (w != nullptr) z = z * r * w[o];
      const float c = inside ? rp.cos[pos * rp.half + pair] : __builtin_nanf("");
      const float sn = inside ? rp.sin[pos * rp.half + pair] : __builtin_nanf("");
      y = first ? y * c - z * sn : y * c + z * sn;
    }
    out[j] = y;
  }
}

template <int TI, int TO>
__global__ __launch_bounds__(256) void k_norm_rope(int64_t tokens, int dim, HeadRows a, HeadRows b, float eps, RopeArgs rp) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int heads = a.heads + b.heads;
  const int64_t t = row / heads;
  if (t >= tokens) return;
  const int h = (int)(row % heads);
  const bool second = h >= a.heads;
  const HeadRows& s = second ? b : a;
  const int hh = second ? h - a.heads : h;
  float y[4];
  head_row<TI>(s.in, t * s.in_token + hh * s.in_head, dim, s.weight, eps, rp, t, lane, y);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j < dim) store1<TO>(s.out, t * s.out_token + hh * s.out_head + lane + 64 * j, y[j]);
}

template <int TI, int TC>
__global__ __launch_bounds__(256) void k_kv_append(int64_t tokens, int dim, HeadRows k, HeadRows v, CacheArgs c,
                                                   const int64_t* slots, float eps, RopeArgs rp) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t t = row / (2 * c.kv_heads);
  if (t >= tokens) return;
  const int h = (int)(row % (2 * c.kv_heads));
  const bool is_v = h >= c.kv_heads;
  const int hh = is_v ? h - c.kv_heads : h;
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= c.n_pages * c.page_size) return;
  const HeadRows& s = is_v ? v : k;
  RopeArgs none;
  float y[4];
  head_row<TI>(s.in, t * s.in_token + hh * s.in_head, dim, s.weight, eps, is_v ? none : rp, t, lane, y);
  const int64_t at = slot / c.page_size * c.page + slot % c.page_size * c.token + hh * c.head;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j < dim) store1<TC>(is_v ? c.v : c.k, at + lane + 64 * j, y[j]);
}

template <class F>
hipError_t by_type(int type, F&& f) {
  switch (type) {
    case DQ_F32: return f(std::integral_constant<int, DQ_F32>{});
    case DQ_F16: return f(std::integral_constant<int, DQ_F16>{});
    default: return f(std::integral_constant<int, DQ_BF16>{});
  }
}

}  // namespace

hipError_t launch_norm_rope(int in_type, int out_type, int64_t tokens, int dim, const HeadRows& a, const HeadRows& b,
                            float eps, const RopeArgs& rope, hipStream_t s) {
  const int64_t blocks = (tokens * (a.heads + b.heads) + 3) / 4;
  return by_type(in_type, [&](auto ti) {
    return by_type(out_type, [&](auto to) {
      hipLaunchKernelGGL((k_norm_rope<ti(), to()>), dim3((uint32_t)blocks), dim3(256), 0, s, tokens, dim, a, b, eps,
                         rope);
      return hipGetLastError();
    });
  });
}

hipError_t launch_kv_append(int in_type, int cache_type, int64_t tokens, int dim, const HeadRows& k, const HeadRows& v,
                            const CacheArgs& cache, const int64_t* slots, float eps, const RopeArgs& rope,
                            hipStream_t s) {
  const int64_t blocks = (tokens * 2 * cache.kv_heads + 3) / 4;
  return by_type(in_type, [&](auto ti) {
    return by_type(cache_type, [&](auto tc) {
      hipLaunchKernelGGL((k_kv_append<ti(), tc()>), dim3((uint32_t)blocks), dim3(256), 0, s, tokens, dim, k, v, cache,
                         slots, eps, rope);
      return hipGetLastError();
    });
  });
}

}  // namespace dq
