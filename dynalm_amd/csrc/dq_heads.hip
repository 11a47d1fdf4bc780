// dq_heads.hip -- norms and rotation of query and key heads, and the append of keys and
// values to a paged cache with both on the way.
//
// A head row is D <= 256 values: y = x / sqrt(mean x^2 + eps) * w, then the first 2 * half of
// them turn in pairs, a' = a c - b s, b' = b c + a s. Every value is read once and written once: the
// bytes are the bound, the launch for a few tokens.
//
// Rows that can be read in 16 bytes take up to 16 lanes each, a lane two chunks of 8 values that hold both
// values of its pairs (chunks j and j + half / 8 for halves, 2j and 2j + 1 for neighbours), so
// that nothing but the sum of squares crosses lanes; a lane's cosines, sines and weights serve several heads of its token
// (k_heads). Other rows take a wave each, value by value (k_norm_rope, k_kv_append): 235 us in place of 37 for 8,192
// tokens of 40 heads, 169 in place of 29 for 16,384 tokens appended.
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

template <int T>
DQ_DEV void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (T == DQ_F32) {
    const v4u* q = reinterpret_cast<const v4u*>(static_cast<const float*>(p) + i);
    const v4u a = q[0], b = q[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = as_f(a[k]), v[4 + k] = as_f(b[k]);
  } else {
    const v4u a = *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = T == DQ_F16 ? h2f(a[k]) : as_f(a[k] << 16);
      v[2 * k + 1] = T == DQ_F16 ? h2f(a[k] >> 16) : as_f(a[k] & 0xFFFF0000u);
    }
  }
}
template <bool kStream>
DQ_DEV void store16(v4u* p, v4u x) {
  if constexpr (kStream)
    __builtin_nontemporal_store(x, p);
  else
    *p = x;
}
template <int T, bool kStream>
DQ_DEV void store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (T == DQ_F32) {
    v4u* q = reinterpret_cast<v4u*>(static_cast<float*>(p) + i);
    store16<kStream>(q, v4u{as_u(v[0]), as_u(v[1]), as_u(v[2]), as_u(v[3])});
    store16<kStream>(q + 1, v4u{as_u(v[4]), as_u(v[5]), as_u(v[6]), as_u(v[7])});
  } else {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    v4u a;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const v2f x = {v[2 * k], v[2 * k + 1]};
      a[k] = T == DQ_F16 ? __builtin_bit_cast(u32, __builtin_convertvector(x, v2h))
                         : __builtin_bit_cast(u32, __builtin_convertvector(x, v2b));
    }
    store16<kStream>(reinterpret_cast<v4u*>(static_cast<uint16_t*>(p) + i), a);
  }
}

// Heads of one token that a lane group takes: a, then b. N heads a group: their cosines, sines and
// weights are read once, and their loads are under way together.
template <int TI, int TO, int N, bool kAppend, bool kStream>
__global__ __launch_bounds__(256) void k_heads(int64_t tokens, int dim, int lanes_log2, HeadRows a, HeadRows b, CacheArgs c,
                                               const int64_t* slots, float eps, RopeArgs rp) {
  const int lanes = 1 << lanes_log2, j = threadIdx.x & (lanes - 1);
  const u32 group = blockIdx.x * (256u >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const u32 na = (a.heads + N - 1) / N, nb = (b.heads + N - 1) / N;
  const int64_t t = group / (na + nb);
  if (t >= tokens) return;
  const u32 part = group % (na + nb);
  const bool second = part >= na;
  const int heads = second ? b.heads : a.heads, h0 = (second ? part - na : part) * N;
  const float* w = second ? b.weight : a.weight;
  const char* in = static_cast<const char*>(second ? b.in : a.in);
  const int64_t in_at = t * (second ? b.in_token : a.in_token), in_head = second ? b.in_head : a.in_head;
  void* out = kAppend ? (void*)(second ? c.v : c.k) : second ? b.out : a.out;
  int64_t out_at = t * (second ? b.out_token : a.out_token), out_head = second ? b.out_head : a.out_head;
  if constexpr (kAppend) {
    const int64_t slot = slots[t];
    if (slot < 0 || slot >= c.n_pages * c.page_size) return;
    out_at = slot / c.page_size * c.page + slot % c.page_size * c.token;
    out_head = c.head;
  }
  const int half = kAppend && second ? 0 : rp.half;  // (values are not rotated)
  // the lane's chunks
  const int chunks = dim / 8, turned = half / 8;
  int ca, cb;
  if (rp.pairs || half == 0) {
    ca = 2 * j;
    cb = 2 * j + 1;
  } else if (j < turned) {
    ca = j;
    cb = j + turned;
  } else {
    ca = 2 * j;  // (2 turned chunks before the first such lane's)
    cb = 2 * j + 1;
  }
  const bool has_a = ca < chunks, has_b = cb < chunks;
  const bool turn_a = 8 * ca < 2 * half, turn_b = 8 * cb < 2 * half;

  float x[N][2][8];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int64_t at = in_at + min(h0 + n, heads - 1) * in_head;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[n][0][i] = x[n][1][i] = 0;
    if (has_a) load8<TI>(in, at + 8 * ca, x[n][0]);
    if (has_b) load8<TI>(in, at + 8 * cb, x[n][1]);
  }
  float cs[8], sn[8];  // of the lane's pairs 8 j .. + 7
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
  if (turn_a) {
    const int64_t pos = rp.positions[t];
    if (pos >= 0 && pos < rp.max_pos) {
      const v4u* pc = reinterpret_cast<const v4u*>(rp.cos + pos * half + 8 * j);
      const v4u* ps = reinterpret_cast<const v4u*>(rp.sin + pos * half + 8 * j);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k == 1 && !turn_b) break;
        const v4u qc = pc[k], qs = ps[k];
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[4 * k + i] = as_f(qc[i]), sn[4 * k + i] = as_f(qs[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < 4 || turn_b) cs[i] = sn[i] = __builtin_nanf("");
    }
  }
  if (w != nullptr) {
    float wa[8], wb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 0;
    if (has_a) load8<DQ_F32>(w, 8 * ca, wa);
    if (has_b) load8<DQ_F32>(w, 8 * cb, wb);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float s = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(x[n][0][i], x[n][0][i], fmaf(x[n][1][i], x[n][1][i], s));
      for (int m = lanes >> 1; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
      const float r = 1.f / sqrtf(s / (float)dim + eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[n][0][i] = x[n][0][i] * r * wa[i];
        x[n][1][i] = x[n][1][i] * r * wb[i];
      }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (h0 + n >= heads) break;
    if (turn_a) {
      if (rp.pairs) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (k == 1 && !turn_b) break;
            const float p = x[n][k][2 * i], q = x[n][k][2 * i + 1];
            x[n][k][2 * i] = p * cs[4 * k + i] - q * sn[4 * k + i];
            x[n][k][2 * i + 1] = q * cs[4 * k + i] + p * sn[4 * k + i];
          }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = x[n][0][i], q = x[n][1][i];
          x[n][0][i] = p * cs[i] - q * sn[i];
          x[n][1][i] = q * cs[i] + p * sn[i];
        }
      }
    }
    const int64_t at = out_at + (h0 + n) * out_head;
    if (has_a) store8<TO, kStream>(out, at + 8 * ca, x[n][0]);
    if (has_b) store8<TO, kStream>(out, at + 8 * cb, x[n][1]);
  }
}

bool aligned16(const void* p, int type, int64_t s0, int64_t s1) {
  const int64_t v = type == DQ_F32 ? 4 : 8;
  return (uintptr_t)p % 16 == 0 && s0 % v == 0 && s1 % v == 0;
}
// Whether a launch's rows, tables and weights can be read and written in 16 bytes, and no chunk of 8
// values holds turned and other ones.
bool in_chunks(int in_type, int out_type, const HeadRows& a, const HeadRows& b, const RopeArgs& rp) {
  for (const HeadRows* r : {&a, &b})
    if (!aligned16(r->in, in_type, r->in_token, r->in_head) || !aligned16(r->out, out_type, r->out_token, r->out_head) ||
        (uintptr_t)r->weight % 16 != 0)
      return false;
  return rp.half == 0 || (rp.half % (rp.pairs ? 4 : 8) == 0 && ((uintptr_t)rp.cos | (uintptr_t)rp.sin) % 16 == 0);
}

// Heads a lane group takes: two once that leaves enough groups for every CU, one below, where latency
// counts; outputs past what the L2s hold (32 MB) are written around them. 8,192 tokens of 40 bf16 heads of 128
// (172 MB moved): 44.0 us with one head, 43.9 with two, 51.6 with four, 61.3 with eight; with
// streaming stores 37.3 (4.6 TB/s) and 41.4 with two and four. 16,384 tokens of 8 + 8 heads appended
// (143 MB): 32.6, 38.4, 39.7, 41.7, and 29.4 (4.85 TB/s) and 31.1. A copy of 1 GiB reaches 4.8 TB/s.
template <int TI, int TO, bool kAppend>
hipError_t launch_heads(int64_t tokens, int dim, const HeadRows& a, const HeadRows& b, const CacheArgs& c,
                        const int64_t* slots, float eps, const RopeArgs& rope, hipStream_t s) {
  int log2 = 0;
  while ((16 << log2) < dim) ++log2;
  const int per = 256 >> log2;
  const int64_t rows = tokens * (a.heads + b.heads);
  const bool many = rows >= 1 << 15, stream = many && rows * dim * (TO == DQ_F32 ? 4 : 2) >= 32 << 20;
  const int n = many ? 2 : 1;
  const int64_t groups = tokens * ((a.heads + n - 1) / n + (b.heads + n - 1) / n);
  const dim3 grid((uint32_t)((groups + per - 1) / per)), block(256);
  if (stream)
    hipLaunchKernelGGL((k_heads<TI, TO, 2, kAppend, true>), grid, block, 0, s, tokens, dim, log2, a, b, c, slots, eps, rope);
  else if (many)
    hipLaunchKernelGGL((k_heads<TI, TO, 2, kAppend, false>), grid, block, 0, s, tokens, dim, log2, a, b, c, slots, eps, rope);
  else
    hipLaunchKernelGGL((k_heads<TI, TO, 1, kAppend, false>), grid, block, 0, s, tokens, dim, log2, a, b, c, slots, eps, rope);
  return hipGetLastError();
}

// A dispatch counts its threads in 32 bits: launches of kLaunchRows head rows at most, of whole tokens, one after
// another (a wave a row, 2^31 threads).
constexpr int64_t kLaunchRows = (int64_t)1 << 25;

// The rows from token t0 on.
HeadRows from_token(HeadRows r, int in_type, int out_type, int64_t t0) {
  r.in = static_cast<const char*>(r.in) + t0 * r.in_token * (in_type == DQ_F32 ? 4 : 2);
  if (r.out != nullptr) r.out = static_cast<char*>(r.out) + t0 * r.out_token * (out_type == DQ_F32 ? 4 : 2);
  return r;
}

// f(first token, tokens) for each launch.
template <class F>
hipError_t by_launch(int64_t tokens, int64_t heads, F&& f) {
  const int64_t most = heads < kLaunchRows ? kLaunchRows / heads : 1;
  for (int64_t t0 = 0; t0 < tokens; t0 += most)
    if (const hipError_t e = f(t0, tokens - t0 < most ? tokens - t0 : most); e != hipSuccess) return e;
  return hipSuccess;
}

template <class F>
hipError_t by_type(int type, F&& f) {
  switch (type) {
    case DQ_F32: return f(std::integral_constant<int, DQ_F32>{});
    case DQ_F16: return f(std::integral_constant<int, DQ_F16>{});
    default: return f(std::integral_constant<int, DQ_BF16>{});
  }
}

template <class F>
hipError_t by_cache_type(int type, F&& f) {
  if (type == DQ_F16) return f(std::integral_constant<int, DQ_F16>{});
  return f(std::integral_constant<int, DQ_BF16>{});
}

}  // namespace

hipError_t launch_norm_rope(int in_type, int out_type, int64_t tokens, int dim, const HeadRows& a, const HeadRows& b,
                            float eps, const RopeArgs& rope, hipStream_t s) {
  const int64_t heads = (int64_t)a.heads + b.heads;
  const bool chunks = in_chunks(in_type, out_type, a, b, rope);
  return by_launch(tokens, heads, [&](int64_t t0, int64_t n) {
    const HeadRows at = from_token(a, in_type, out_type, t0), bt = from_token(b, in_type, out_type, t0);
    RopeArgs rt = rope;
    if (rt.positions != nullptr) rt.positions += t0;
    return by_type(in_type, [&](auto ti) {
      return by_type(out_type, [&](auto to) {
        if (chunks) return launch_heads<ti(), to(), false>(n, dim, at, bt, CacheArgs{}, nullptr, eps, rt, s);
        hipLaunchKernelGGL((k_norm_rope<ti(), to()>), dim3((uint32_t)((n * heads + 3) / 4)), dim3(256), 0, s, n, dim, at,
                           bt, eps, rt);
        return hipGetLastError();
      });
    });
  });
}

hipError_t launch_kv_append(int in_type, int cache_type, int64_t tokens, int dim, const HeadRows& k, const HeadRows& v,
                            const CacheArgs& cache, const int64_t* slots, float eps, const RopeArgs& rope,
                            hipStream_t s) {
  const int64_t heads = 2 * (int64_t)cache.kv_heads;
  const bool chunks = in_chunks(in_type, cache_type, k, v, rope);  // (the cache's places are 16-byte aligned always)
  return by_launch(tokens, heads, [&](int64_t t0, int64_t n) {
    const HeadRows kt = from_token(k, in_type, cache_type, t0), vt = from_token(v, in_type, cache_type, t0);
    RopeArgs rt = rope;
    if (rt.positions != nullptr) rt.positions += t0;
    return by_type(in_type, [&](auto ti) {
      return by_cache_type(cache_type, [&](auto tc) {
        if (chunks) return launch_heads<ti(), tc(), true>(n, dim, kt, vt, cache, slots + t0, eps, rt, s);
        hipLaunchKernelGGL((k_kv_append<ti(), tc()>), dim3((uint32_t)((n * heads + 3) / 4)), dim3(256), 0, s, n, dim, kt,
                           vt, cache, slots + t0, eps, rt);
        return hipGetLastError();
      });
    });
  });
}

}  // namespace dq
