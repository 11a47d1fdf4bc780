// dq_attn.hip -- attention of a batch over a shared prefix and each sequence's own pages.
#include <type_traits>

#include "dq_attn.h"
#include "dq_device.h"

namespace dq {
namespace {

template <int T>
DQ_DEV float widen(u32 h) {
  if constexpr (T == DQ_F16) return h2f(h);
  return as_f(h << 16);
}
template <int T>
DQ_DEV float load1(const void* p, int64_t i) {
  if constexpr (T == DQ_F32) return static_cast<const float*>(p)[i];
  return widen<T>(static_cast<const uint16_t*>(p)[i]);
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

// The sequence of token t: the last b with q_offsets[b] <= t (-1: none), its first token and count.
struct Seq {
  int b, first, n;
};
DQ_DEV Seq find_seq(const AttnArgs& a, int t) {
  if (a.q_offsets == nullptr) return Seq{t, t, 1};
  int lo = -1, hi = a.batch;  // q_offsets[lo] <= t < q_offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.q_offsets[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  if (lo < 0) return Seq{-1, 0, 0};
  const int first = a.q_offsets[lo], end = a.q_offsets[lo + 1];
  return t < end ? Seq{lo, first, end - first} : Seq{-1, 0, 0};
}

// One wave a query row: 64 keys at a time, a lane each for the scores, then lanes over the
// head's values for the sum of v.
template <int T, int TC>
__global__ __launch_bounds__(64) void k_attn_rows(AttnArgs a) {
  __shared__ float qs[DQ_MAX_HEAD_DIM];
  __shared__ float ps[64];
  __shared__ int64_t at[64];
  const int lane = threadIdx.x;
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const Seq sq = find_seq(a, t);
  if (sq.b < 0) return;
  const int len = a.max_len > 0 ? min(max(a.lens[sq.b], 0), a.max_len) : 0;
  const int own = min(max(len - sq.n + (t - sq.first) + 1, 0), len);
  for (int d = lane; d < a.dim; d += 64) qs[d] = load1<T>(a.q, t * a.q_token + h * a.q_head + d);
  __syncthreads();
  const int hk = h / a.group;
  const CacheArgs& c = a.cache;
  float m = -INFINITY, l = 0, o[4] = {0, 0, 0, 0};
  bool bad = false;
  for (int part = 0; part < 2; ++part) {
    const int keys = part == 0 ? a.prefix_len : own;
    const int32_t* pages = part == 0 ? a.prefix_pages : a.pages + sq.b * a.pages_stride;
    for (int j0 = 0; j0 < keys; j0 += 64) {
      const int j = j0 + lane, cnt = min(64, keys - j0);
      float s = -INFINITY;
      if (j < keys) {
        int id = pages[j / c.page_size];
        if (id < 0 || id >= c.n_pages) {
          bad = true;
          id = 0;
        }
        const int64_t off = id * c.page + j % c.page_size * c.token + hk * c.head;
        at[lane] = off;
        float acc = 0;
        for (int d = 0; c.n_pages > 0 && d < a.dim; ++d) acc = fmaf(qs[d], widen<TC>(c.k[off + d]), acc);
        s = acc * a.scale_log2;
      }
      float mx = s;
      for (int k = 32; k >= 1; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
      mx = fmaxf(mx, m);
      const float base = mx == -INFINITY ? 0.f : mx;
      const float p = j < keys ? exp2f(s - base) : 0.f, alpha = exp2f(m - base);
      float sum = p;
      for (int k = 32; k >= 1; k >>= 1) sum += __shfl_xor(sum, k, 64);
      l = l * alpha + sum;
      m = mx;
      ps[lane] = p;
      __syncthreads();
      for (int i = 0; i < 4; ++i) o[i] *= alpha;
      for (int k = 0; c.n_pages > 0 && k < cnt; ++k)
        for (int i = 0; i < 4; ++i)
          if (lane + 64 * i < a.dim) o[i] = fmaf(ps[k], widen<TC>(c.v[at[k] + lane + 64 * i]), o[i]);
      __syncthreads();
    }
  }
  const bool nan = __any(bad);
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.dim) {
      const float y = nan ? __builtin_nanf("") : l == 0.f ? 0.f : o[i] / l;
      store1<T>(a.out, t * a.out_token + h * a.out_head + lane + 64 * i, y);
    }
  if (a.lse != nullptr && lane == 0)
    a.lse[(int64_t)t * a.heads + h] = nan ? __builtin_nanf("") : l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718f;
}

template <int T, int TC>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_attn_rows<T, TC>), dim3((uint32_t)(a.tokens * a.heads)), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(int type, int cache_type, const AttnArgs& a, hipStream_t s) {
  if (cache_type == DQ_F16) return type == DQ_F32 ? launch<DQ_F32, DQ_F16>(a, s) : launch<DQ_F16, DQ_F16>(a, s);
  return type == DQ_F32 ? launch<DQ_F32, DQ_BF16>(a, s) : launch<DQ_BF16, DQ_BF16>(a, s);
}

}  // namespace dq
