// dq_attn_device.h -- device helpers that the attention kernels share: number types, the 16-bit
// matrix instruction, the softmax's running maximum, query operands, rows and their sequences.
#pragma once

#include "dq_attn.h"
#include "dq_device.h"

namespace dq {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));

template <int T>
DQ_DEV float widen(u32 h) {
  if constexpr (T == DQ_F16) return h2f(h);
  return as_f(h << 16);
}
template <int T>
DQ_DEV float widen_hi(u32 h) {
  if constexpr (T == DQ_F16) return h2f(h >> 16);
  return as_f(h & 0xFFFF0000u);
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
// Two floats to the nearest values of type T, a in the low half.
template <int T>
DQ_DEV u32 pack(float a, float b) {
  if constexpr (T == DQ_F16) return __builtin_bit_cast(u32, __builtin_convertvector(v2f{a, b}, v2h));
  return __builtin_bit_cast(u32, __builtin_convertvector(v2f{a, b}, v2b));
}

// Parts that an fp32 operand is split into beside a cache of type TC: two f16 parts hold 22 bits
// (of rows scaled to f16's range), three bf16 parts all 24. A 16-bit operand is its only part.
template <int T, int TC>
constexpr int kParts = T != DQ_F32 ? 1 : TC == DQ_F16 ? 2 : 3;

template <int T, int TC>
DQ_DEV void split(float a, float b, u32 (&out)[kParts<T, TC>]) {
  out[0] = pack<TC>(a, b);
#pragma unroll
  for (int i = 1; i < kParts<T, TC>; ++i) {
    a -= widen<TC>(out[i - 1]);
    b -= widen_hi<TC>(out[i - 1]);
    out[i] = pack<TC>(a, b);
  }
}

// The running maximum m of a row moves only when a score passes it by more than kSlack (in powers of
// two), so that the sums are seldom rescaled; weights run as 2^(s - m + kShift), at most 2^14: f16 weights
// far below the largest stay normal numbers (what l and O share cancels).
constexpr float kSlack = 8.f;
template <int TC>
constexpr float kShift = TC == DQ_F16 ? 6.f : 0.f;

// C + A . B over a 16 x 16 x 32 tile: lane l supplies row (A) / column (B) l % 16 and K = 8 (l / 16)
// .. + 7; it holds column l % 16, rows 4 (l / 16) .. + 3 of C.
template <int TC>
DQ_DEV v4f mma(v4u a, v4u b, v4f c) {
  if constexpr (TC == DQ_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

DQ_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32: within an ulp

// The largest (the sum) over the four lane groups that hold one row.
DQ_DEV float row_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(as_u(x), as_u(x), false, false);
  x = fmaxf(as_f(a[0]), as_f(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(as_u(x), as_u(x), false, false);
  return fmaxf(as_f(b[0]), as_f(b[1]));
}
DQ_DEV float row_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(as_u(x), as_u(x), false, false);
  x = as_f(a[0]) + as_f(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(as_u(x), as_u(x), false, false);
  return as_f(b[0]) + as_f(b[1]);
}

// The least over a wave.
DQ_DEV u32 wave_least(u32 x) {
  x = min(x, (u32)dpp<kQuadXor1>((int)x));
  x = min(x, (u32)dpp<kQuadXor2>((int)x));
  x = min(x, (u32)dpp<kHalfMirror>((int)x));
  x = min(x, (u32)dpp<kRowRor8>((int)x));
  auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = min((u32)a[0], (u32)a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return min((u32)b[0], (u32)b[1]);
}

// Every load of the wave has come.
DQ_DEV void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}

// A page number through the scalar cache.
DQ_DEV int page_at(const int32_t* pages, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)pages)[i];
}

template <int TC>
constexpr u32 kExp = TC == DQ_F16 ? 0x7C00u : 0x7F80u;

template <int TC>
DQ_DEV bool nonfinite(u32 x) {
  return (x & kExp<TC>) == kExp<TC> || (x & (kExp<TC> << 16)) == (kExp<TC> << 16);
}

DQ_DEV int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Eight values of q from each of the values `at` on, all under way together.
template <int T, int N>
DQ_DEV void load8s(const AttnArgs& a, const int64_t (&at)[N], v4u (&x)[N][T == DQ_F32 ? 2 : 1]) {
  constexpr int kBytes = T == DQ_F32 ? 4 : 2;
  if (a.q_vec) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int k = 0; k < (T == DQ_F32 ? 2 : 1); ++k) x[n][k] = reinterpret_cast<const v4u*>(static_cast<const char*>(a.q) + at[n] * kBytes)[k];
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const char* p = static_cast<const char*>(a.q) + at[n] * kBytes;
#pragma unroll
      for (int i = 0; i < (T == DQ_F32 ? 8 : 4); ++i)
        x[n][i / 4][i % 4] = T == DQ_F32 ? reinterpret_cast<const u32*>(p)[i]
                                         : (u32)reinterpret_cast<const uint16_t*>(p)[2 * i] | (u32)reinterpret_cast<const uint16_t*>(p)[2 * i + 1] << 16;
    }
  }
}

// The query fragments of rows: lane l has row l % 16 and, of every 32 values, 8 (l / 16) .. + 7. First their loads,
// then, once other loads are under way too, the operands; the latter returns
// the factor from products to scores in powers of two: fp32 rows are scaled to a largest value
// in [2^14, 2^15), where all of their parts are normal numbers.
template <int T, int DP>
struct RawQ {
  v4u x[DP / 32][T == DQ_F32 ? 2 : 1];
};
// 16 bytes of them: from value d of the head, in fp32 its values 4 k .. + 3 of 8 (0 past the head's dimension).
template <int T>
DQ_DEV v4u load_q16(const AttnArgs& a, int token, int head, int d, int k) {
  const int64_t at = (int64_t)token * a.q_token + (int64_t)head * a.q_head + d;
  v4u x = {0, 0, 0, 0};
  if (d < a.dim) {
    if constexpr (T == DQ_F32) {
      const float* p = static_cast<const float*>(a.q) + at + 4 * k;
      if (a.q_vec)
        x = *reinterpret_cast<const v4u*>(p);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = as_u(p[i]);
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(a.q) + at;
      if (a.q_vec)
        x = *reinterpret_cast<const v4u*>(p);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (u32)p[2 * i] | ((u32)p[2 * i + 1] << 16);
    }
  }
  return x;
}
template <int T, int DP>
DQ_DEV void load_q(const AttnArgs& a, bool valid, int token, int head, int g, RawQ<T, DP>& r) {
#pragma unroll
  for (int s = 0; s < DP / 32; ++s)
#pragma unroll
    for (int k = 0; k < (T == DQ_F32 ? 2 : 1); ++k) r.x[s][k] = valid ? load_q16<T>(a, token, head, 32 * s + 8 * g, k) : v4u{0, 0, 0, 0};
}
template <int T, int TC, int DP>
DQ_DEV float q_operands(const AttnArgs& a, const RawQ<T, DP>& r, v4u (&q)[kParts<T, TC>][DP / 32]) {
  if constexpr (T != DQ_F32) {
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) q[0][s] = r.x[s][0];
    return a.scale_log2;
  } else {
    float most = 0;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(as_f(r.x[s][i / 4][i % 4])));
    most = row_max(most);
    const int e = most > 0 && most < INFINITY ? 15 - (__builtin_amdgcn_frexp_expf(most)) : 0;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32 parts[kParts<T, TC>];
        split<T, TC>(ldexpf(as_f(r.x[s][i / 2][i % 2 * 2]), e), ldexpf(as_f(r.x[s][i / 2][i % 2 * 2 + 1]), e), parts);
#pragma unroll
        for (int k = 0; k < kParts<T, TC>; ++k) q[k][s][i] = parts[k];
      }
    return fmaxf(ldexpf(a.scale_log2, -e), 1.2e-38f);  // (0 would make NaN of a masked score)
  }
}

DQ_DEV float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));  // (fmaxf would quieten each operand first)
  return r;
}

// A row's running maximum m and the base that its weights are taken from.
struct RowMax {
  float m = -INFINITY, base = 0;
};

// Whether one of the lane's N products x passes its row's maximum.
template <int N>
DQ_DEV bool passes(const float (&x)[N], float c, const RowMax& r, float& mx) {
  mx = max3(x[0], x[1], x[2]);
#pragma unroll
  for (int i = 3; i + 1 < N; i += 2) mx = max3(mx, x[i], x[i + 1]);
  if (N % 2 == 0) mx = fmaxf(mx, x[N - 1]);
  return mx * c > r.m + kSlack;
}
// Moves the maximum of the rows that are passed (mx: the lane's largest product) and returns the
// factor of what was summed before; a row does not move for another.
template <int TC>
DQ_DEV float move_max(float mx, float c, RowMax& r) {
  mx = row_max(mx) * c;
  if (!(mx > r.m + kSlack)) return 1.f;
  const float alpha = exp2_fast(r.m - mx);
  r.m = mx;
  r.base = mx - kShift<TC>;
  return alpha;
}

// Four values of a row from value d on: finished (o / l) or as they are into the workspace.
template <int T>
DQ_DEV void store4(const AttnArgs& a, int64_t at, int d, v4f y) {
  if (a.out_vec) {
    if constexpr (T == DQ_F32)
      *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + at + d) = y;
    else
      *reinterpret_cast<v2u*>(static_cast<uint16_t*>(a.out) + at + d) = v2u{pack<T>(y[0], y[1]), pack<T>(y[2], y[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) store1<T>(a.out, at + d + i, y[i]);
  }
}

// The finished values of a row: zeros where no weight was above zero (whatever infinite or NaN values it saw).
DQ_DEV v4f finish(v4f o, float sum, float inv) {
  v4f y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = sum == 0.f ? 0.f : o[i] * inv;
  return y;
}

DQ_DEV float lse_of(float m, float l, float shift) {
  return l == 0.f ? -INFINITY : (float)(((double)(m - shift) + (double)__log2f(l)) * 0.693147180559945309);
}

// A sequence's keys, whatever its length holds.
DQ_DEV int seq_len(const AttnArgs& a, int b) { return a.max_len > 0 ? min(max(a.lens[b], 0), a.max_len) : 0; }

// The sequence of token t, the last b with q_offsets[b] <= t (-1: none): a wave's lanes look at 64 places
// at a time.
DQ_DEV int find_seq(const AttnArgs& a, int t, int lane) {
  if (a.q_offsets == nullptr) return t;
  int lo = 0, n = a.batch + 1;  // entries still in question: the count of those <= t is in lo .. lo + n
  while (n > 0) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const bool le = lane * step < n && a.q_offsets[i] <= t;
    const int cnt = __popcll(__ballot(le));
    if (cnt == 0) break;
    if (step == 1) {
      lo += cnt;
      break;
    }
    const int last = (cnt - 1) * step;  // entry lo + last is <= t, the next looked at is not
    n = min(step, n - last) - 1;
    lo += last + 1;
  }
  lo = uniform(lo);
  return lo >= 1 && lo <= a.batch ? lo - 1 : -1;
}

}  // namespace
}  // namespace dq
