// dq_attn.hip -- attention of a batch over a shared prefix and each sequence's own pages.
//
// For a query row q and its visible keys k_j: s_j = scale q . k_j, o = sum_j e^(s_j - m) v_j /
// sum_j e^(s_j - m), in one pass with a running maximum m. Both products run on the 16-bit matrix
// cores over tiles of 16 rows (v_mfma_f32_16x16x32): S^T = K Q^T leaves a lane with one row's
// scores of four consecutive keys, which is, after the exponential, the operand that O^T = V^T P^T
// takes: the weights never leave their lane. Which key a K-slot of the second product holds is
// free as long as both operands agree: slot 8 g + j of a lane group g is key 16 (j / 4) + 4 g +
// j % 4 of 32.
//
// The work is split in items of (kv head, row tile, key range). Rows of one kv head are its
// `group` query heads times the tokens, so that a key is read once for all of them; the prefix
// takes the rows of the whole batch together, the own keys those of one sequence. Ranges of a
// row that run in several items leave (O, m, l) in the workspace and k_attn_join adds them.
#include <type_traits>

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

#define DQ_LDS(T) __attribute__((address_space(3))) T

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

// The weights run as 2^(s - m + kShift): f16 weights far below the largest stay normal numbers
// (2^14 is the largest; what l and O share cancels).
template <int TC>
constexpr float kShift = TC == DQ_F16 ? 14.f : 0.f;

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

// ---- infinite and NaN values that only some rows of a tile see ------------
// A masked key has weight 0, but 0 times an infinite value is NaN in a matrix product. In tiles
// that some rows see in part, such values are taken out of the product and added to the rows that
// see them.
template <int TC>
constexpr u32 kExp = TC == DQ_F16 ? 0x7C00u : 0x7F80u;
template <int TC>
constexpr u32 kOne = TC == DQ_F16 ? 0x3C00u : 0x3F80u;

template <int TC>
DQ_DEV bool has_nonfinite(v4u x) {
  bool nf = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    nf |= (x[i] & kExp<TC>) == kExp<TC> || (x[i] & (kExp<TC> << 16)) == (kExp<TC> << 16);
  return nf;
}
template <int TC>
DQ_DEV void take_nonfinite(v4u& x, v4u& pos, v4u& neg) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32 c = 0, p = 0, n = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32 v = (x[i] >> (16 * h)) & 0xFFFFu;
      const bool nf = (v & kExp<TC>) == kExp<TC>, nan = nf && (v & 0x7FFFu) != kExp<TC>, sign = v >> 15;
      c |= (nf ? 0u : v) << (16 * h);
      p |= (nf && (nan || !sign) ? kOne<TC> : 0u) << (16 * h);
      n |= (nf && (nan || sign) ? kOne<TC> : 0u) << (16 * h);
    }
    x[i] = c;
    pos[i] = p;
    neg[i] = n;
  }
}
template <int TC>
DQ_DEV v4f add_nonfinite(v4u pos, v4u neg, v4u sees, v4f o) {
  const v4f p = mma<TC>(pos, sees, v4f{0, 0, 0, 0}), n = mma<TC>(neg, sees, v4f{0, 0, 0, 0});
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] += (p[i] > 0 ? INFINITY : 0.f) + (n[i] > 0 ? -INFINITY : 0.f);
  return o;
}

// ---- rows ------------------------------------------------------------------

DQ_DEV int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The rows of an item: `count` of them from row `first` of kv head `head`'s rows (row = token * group
// + query head of the group), and the keys that they see: all of the prefix, and own keys below
// own0 + (token - token0), at most len.
struct Item {
  int head, first, count;
  int token0, own0, len;
  int b;             // the sequence (-1: rows of all)
  int pk0, pk1;      // range of the prefix
  int ok0, ok1;      // range of the own keys
  int slot;
};

// This workgroup's item; false where there is none. `tile`: rows of a tile.
DQ_DEV bool find_item(const AttnArgs& a, const AttnPart& w, bool stacked, int index, int tile, Item& it) {
  const int hk = a.cache.kv_heads;
  const int t = index % w.tiles;
  int rest = index / w.tiles;
  it.head = rest % hk;
  rest /= hk;
  const int split = rest % w.splits;
  it.slot = w.slot + split;
  const int k0 = split * w.chunk, k1 = k0 + w.chunk;
  it.pk0 = it.pk1 = it.ok0 = it.ok1 = 0;
  if (stacked) {
    it.b = -1;
    it.first = t * tile;
    it.count = min(tile, a.tokens * a.group - it.first);
    it.token0 = it.own0 = it.len = 0;
    it.pk0 = k0;
    it.pk1 = min(k1, a.prefix_len);
    return true;
  }
  const int b = rest / w.splits;
  it.b = b;
  const int lo = a.q_offsets != nullptr ? a.q_offsets[b] : b;
  const int hi = a.q_offsets != nullptr ? a.q_offsets[b + 1] : b + 1;
  // (whatever the offsets hold, rows stay inside the tensors)
  const int first = min(max(lo, 0), a.tokens);
  const int n = min(min(max(hi, first), a.tokens) - first, a.max_q);
  const int tt = w.backward ? w.tiles - 1 - t : t;
  it.count = min(tile, n * a.group - tt * tile);
  if (it.count <= 0) return false;
  it.first = first * a.group + tt * tile;
  it.len = a.max_len > 0 ? min(max(a.lens[b], 0), a.max_len) : 0;
  it.token0 = first;
  it.own0 = it.len - n + 1;
  if (w.with_prefix) {  // prefix, then (from the next whole chunk unit on) own keys
    const int gap = w.own_from;
    it.pk0 = min(k0, a.prefix_len);
    it.pk1 = min(k1, a.prefix_len);
    it.ok0 = max(k0 - gap, 0);
    it.ok1 = min(max(k1 - gap, 0), it.len);
  } else {
    it.ok0 = k0;
    it.ok1 = min(k1, it.len);
  }
  // the last row sees the most
  const int most = min(max(it.own0 + (it.first + it.count - 1) / a.group - first, 0), it.len);
  it.ok1 = min(it.ok1, most);
  if (split > 0 && it.pk0 >= it.pk1 && k0 - (w.with_prefix ? w.own_from : 0) >= it.len) return false;  // past the sequence: the join leaves it out
  return true;
}

// Own keys that row r sees.
DQ_DEV int own_limit(const AttnArgs& a, const Item& it, int token) {
  return it.b < 0 ? 0 : min(max(it.own0 + token - it.token0, 0), it.len);
}

// The query fragments of rows: lane l has row l % 16 and, of every 32 values, 8 (l / 16) .. + 7. Returns
// the factor from products to scores in powers of two: fp32 rows are scaled to a largest value
// in [2^14, 2^15), where all of their parts are normal numbers.
template <int T, int TC, int DP>
DQ_DEV float load_q(const AttnArgs& a, bool valid, int token, int head, int g, v4u (&q)[kParts<T, TC>][DP / 32]) {
  const int64_t base = (int64_t)token * a.q_token + (int64_t)head * a.q_head;
  if constexpr (T != DQ_F32) {
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + base;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
      const int d = 32 * s + 8 * g;
      v4u x = {0, 0, 0, 0};
      if (valid && d < a.dim) {
        if (a.q_vec)
          x = *reinterpret_cast<const v4u*>(p + d);
        else
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = (u32)p[d + 2 * i] | ((u32)p[d + 2 * i + 1] << 16);
      }
      q[0][s] = x;
    }
    return a.scale_log2;
  } else {
    const float* p = static_cast<const float*>(a.q) + base;
    float x[DP / 32][8];
    float most = 0;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
      const int d = 32 * s + 8 * g;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = 0;
      if (valid && d < a.dim) {
        if (a.q_vec) {
          const v4f lo = *reinterpret_cast<const v4f*>(p + d), hi = *reinterpret_cast<const v4f*>(p + d + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][i] = lo[i], x[s][4 + i] = hi[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[s][i] = p[d + i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[s][i]));
    }
    most = row_max(most);
    const int e = most > 0 && most < INFINITY ? 15 - (__builtin_amdgcn_frexp_expf(most)) : 0;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32 parts[kParts<T, TC>];
        split<T, TC>(ldexpf(x[s][2 * i], e), ldexpf(x[s][2 * i + 1], e), parts);
#pragma unroll
        for (int k = 0; k < kParts<T, TC>; ++k) q[k][s][i] = parts[k];
      }
    return fmaxf(ldexpf(a.scale_log2, -e), 1.2e-38f);  // (0 would make NaN of a masked score)
  }
}

// One step of a row's running maximum over N scores a lane (products x, which become weights):
// returns the factor of what was summed before.
template <int TC, int N>
DQ_DEV float softmax_step(float (&x)[N], float c, float& m, float& l) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmaxf(mx, x[i]);
  mx = fmaxf(m, row_max(mx) * c);
  const float base = mx == -INFINITY ? 0.f : mx - kShift<TC>;
  const float alpha = m == mx ? 1.f : exp2_fast(m - mx);
  float sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = exp2_fast(fmaf(x[i], c, -base));
    sum += x[i];
  }
  l = fmaf(l, alpha, sum);
  m = mx;
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

DQ_DEV float lse_of(float m, float l, float shift) {
  return l == 0.f ? -INFINITY : (float)(((double)(m - shift) + (double)__log2f(l)) * 0.693147180559945309);
}

// ---- few rows: up to 16 of one item ----------------------------------------
// The four waves take 32 keys each in turn, with a running softmax of their own, and add up at
// the end: a decode step's own keys, where a tile of 16 rows is mostly empty and the keys' bytes
// are all that counts. Keys and values go straight from memory to registers: a lane's 16 bytes of a key
// are its A operand as they lie; of the values it takes DP / 16 of 8 keys, which v_perm turns into
// the operands of DP / 16 tiles.

template <int DP>
struct KvRegs {
  v4u k[2][DP / 32];
  u32 v[8][DP / 32];  // [key slot][dword]: DP / 16 values
};

template <int T, int TC, int DP>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_attn_few(AttnArgs a, AttnPart w, bool stacked) {
  constexpr int NP = kParts<T, TC>;
  constexpr int NC = DP / 16;
  __shared__ float s_ml[4][16][2];
  __shared__ v4f s_o[4][16][DP / 4];
  __shared__ int s_bad;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  Item it;
  if (!find_item(a, w, stacked, blockIdx.x, 16, it)) return;
  if (threadIdx.x == 0) s_bad = 0;

  const bool valid = n < it.count;
  const int row = it.first + (valid ? n : 0);
  const int token = row / a.group, qh = it.head * a.group + row % a.group;
  const int own_lim = own_limit(a, it, token);
  const int own_least = own_limit(a, it, it.first / a.group);
  v4u q[NP][DP / 32];
  const float c = load_q<T, TC, DP>(a, valid, token, qh, g, q);

  float m = -INFINITY, l = 0;
  v4f o[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i] = v4f{0, 0, 0, 0};
  bool bad = false;

  const CacheArgs& ca = a.cache;
  const u32 token_bytes = (u32)ca.token * 2;
  constexpr u32 kOut = 0x80000000u;  // an offset past every buffer: such loads give 0
  u32 koff[DP / 32], voff[DP / 128 > 0 ? DP / 128 : 1];
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) koff[s] = 32 * s + 8 * g < a.dim ? n * token_bytes + (32 * s + 8 * g) * 2 : kOut;
#pragma unroll
  for (int s = 0; s < (DP / 128 > 0 ? DP / 128 : 1); ++s) {
    const int d = n * NC + 8 * s;
    voff[s] = d < a.dim ? 4 * g * token_bytes + d * 2 : kOut;
  }

  auto base_of = [&](const int32_t* pages, int key) -> int64_t {
    const int p = key / ca.page_size;
    int id = uniform(pages[p]);
    if ((u32)id >= (u32)ca.n_pages) {
      bad = true;
      id = 0;
    }
    return (int64_t)id * ca.page + (int64_t)(key - p * ca.page_size) * ca.token + (int64_t)it.head * ca.head;
  };
  auto load = [&](const int32_t* pages, int kb, int kend, KvRegs<DP>& r) {
    int64_t base[2];
    base[0] = base_of(pages, kb);
    base[1] = kb + 16 < kend ? base_of(pages, kb + 16) : base[0];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const auto kr = rsrc(ca.k + base[t], 0x7FFFFFFFu);
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) r.k[t][s] = ld16(kr, koff[s]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const auto vr = rsrc(ca.v + base[t], 0x7FFFFFFFu);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DP == 64) {
          const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(vr, voff[0], i * token_bytes, 0));
          r.v[4 * t + i][0] = x[0];
          r.v[4 * t + i][1] = x[1];
        } else {
#pragma unroll
          for (int s = 0; s < DP / 128; ++s) {
            const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[s], i * token_bytes, 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) r.v[4 * t + i][4 * s + e] = x[e];
          }
        }
      }
    }
  };
  auto compute = [&](int kb, int kend, int lim, int least, KvRegs<DP>& r) {
    float x[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      v4f acc = {0, 0, 0, 0};
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) acc = mma<TC>(r.k[t][s], q[p][s], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * t + i] = acc[i];
    }
    const bool edge = kb + 32 > least || kb + 32 > kend;
    v4u sees = {0, 0, 0, 0};
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool in = key < lim && key < kend;
        x[j] = in ? x[j] : -INFINITY;
        sees[j >> 1] |= in ? kOne<TC> << (16 * (j & 1)) : 0u;
        if (key >= kend)  // places past the keys may hold anything
#pragma unroll
          for (int e = 0; e < DP / 32; ++e) r.v[j][e] = 0;
      }
    }
    const float alpha = softmax_step<TC, 8>(x, c, m, l);
    v4u p[NP];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32 parts[NP];
      split<T, TC>(x[2 * j], x[2 * j + 1], parts);
#pragma unroll
      for (int k = 0; k < NP; ++k) p[k][j] = parts[k];
    }
    if (__any(alpha != 1.f)) {
#pragma unroll
      for (int i = 0; i < NC; ++i) o[i] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      v4u vt;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vt[e] = __builtin_amdgcn_perm(r.v[2 * e + 1][i >> 1], r.v[2 * e][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
      if (edge && __any(has_nonfinite<TC>(vt))) {
        v4u pos, neg;
        take_nonfinite<TC>(vt, pos, neg);
        o[i] = add_nonfinite<TC>(pos, neg, sees, o[i]);
      }
#pragma unroll
      for (int k = NP - 1; k >= 0; --k) o[i] = mma<TC>(vt, p[k], o[i]);
    }
  };
  auto range = [&](const int32_t* pages, int k0, int k1, int lim, int least) {
    int kb = k0 + 32 * wave;
    if (kb >= k1) return;
    if constexpr (DP <= 128) {
      KvRegs<DP> r0, r1;
      load(pages, kb, k1, r0);
      while (true) {
        if (kb + 128 < k1) load(pages, kb + 128, k1, r1);
        compute(kb, k1, lim, least, r0);
        kb += 128;
        if (kb >= k1) break;
        if (kb + 128 < k1) load(pages, kb + 128, k1, r0);
        compute(kb, k1, lim, least, r1);
        kb += 128;
        if (kb >= k1) break;
      }
    } else {
      for (; kb < k1; kb += 128) {
        KvRegs<DP> r;
        load(pages, kb, k1, r);
        compute(kb, k1, lim, least, r);
      }
    }
  };
  range(a.prefix_pages, it.pk0, it.pk1, valid ? it.pk1 : 0, it.pk1);
  if (it.b >= 0) range(a.pages + it.b * a.pages_stride, it.ok0, it.ok1, valid ? own_lim : 0, own_least);

  // the waves' sums join in LDS
  l = row_sum(l);
  if (g == 0) {
    s_ml[wave][n][0] = m;
    s_ml[wave][n][1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = (4 * g + i) * NC;
#pragma unroll
    for (int e = 0; e < NC / 4; ++e) s_o[wave][n][d / 4 + e] = v4f{o[4 * e][i], o[4 * e + 1][i], o[4 * e + 2][i], o[4 * e + 3][i]};
  }
  __syncthreads();
  if (bad) s_bad = 1;
  __syncthreads();
  const int quads = a.dim / 4;
  for (int i = threadIdx.x; i < it.count * quads; i += 256) {
    const int r = i / quads, d4 = i % quads;
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) mx = fmaxf(mx, s_ml[k][r][0]);
    v4f y = {0, 0, 0, 0};
    float sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float mk = s_ml[k][r][0];
      const float f = mk == -INFINITY ? 0.f : exp2_fast(mk - mx);
      sum = fmaf(s_ml[k][r][1], f, sum);
      if (mk != -INFINITY) y += s_o[k][r][d4] * f;
    }
    if (s_bad) sum = __builtin_nanf("");
    const int rw = it.first + r, tk = rw / a.group, h = it.head * a.group + rw % a.group;
    if (a.part_o == nullptr) {
      if (it.b < 0 && a.q_offsets != nullptr && (tk < a.q_offsets[0] || tk >= a.q_offsets[a.batch])) continue;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      store4<T>(a, (int64_t)tk * a.out_token + (int64_t)h * a.out_head, 4 * d4, y * inv);
      if (a.lse != nullptr && d4 == 0) a.lse[(int64_t)tk * a.heads + h] = lse_of(mx, sum, kShift<TC>);
    } else {
      const int64_t at = ((int64_t)it.slot * ca.kv_heads + it.head) * a.tokens * a.group + rw;
      *reinterpret_cast<v4f*>(a.part_o + at * a.dim + 4 * d4) = y;
      if (d4 == 0) *reinterpret_cast<v2f*>(a.part_ml + at * 2) = v2f{mx, sum};
    }
  }
}

// ---- many rows: tiles of 64 RT rows ------------------------------------------
// Each wave owns 16 RT rows; the workgroup shares tiles of KT keys and values in LDS, two
// buffers deep, filled by loads that go straight to LDS (a lane's 16 bytes land at 16 times its
// number, so the order of a row's 16-byte chunks is chosen on the reading side: a chunk's place
// is its number XOR a few bits of its key, which spreads a column of keys over all banks). Keys are
// read as A operands, values transposed on the way (ds_read_b64_tr_b16: a lane group's 16 lanes
// read 4 keys x 16 values and each receives one value of the 4 keys).

template <int DP>
constexpr int kTileKeys = DP <= 128 ? 64 : 32;

template <int DP>
DQ_DEV int swizzle_k(int key) {
  return DP == 64 ? (key >> 1) & 7 : key & 15;
}
template <int DP>
DQ_DEV int swizzle_v(int key) {
  return DP == 64 ? ((key >> 1) & 3) << 1 : (key & 7) << 1;
}

template <int T, int TC, int DP, int RT>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_attn_tile(AttnArgs a, AttnPart w, bool stacked) {
  constexpr int NP = kParts<T, TC>;
  constexpr int NC = DP / 16, KT = kTileKeys<DP>, CH = DP / 8;
  constexpr int KW = KT / 4, KI = 64 / CH;  // keys a wave loads of a tile, and with one instruction
  __shared__ __align__(16) uint16_t s_k[2][KT * DP];
  __shared__ __align__(16) uint16_t s_v[2][KT * DP];
  __shared__ int s_bad;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  Item it;
  if (!find_item(a, w, stacked, blockIdx.x, 64 * RT, it)) return;
  if (threadIdx.x == 0) s_bad = 0;
  if (a.dim < DP) {  // the loads leave the places past a head's values as they are: zero
    for (int i = threadIdx.x; i < 2 * KT * DP / 8; i += 256) {
      reinterpret_cast<v4u*>(&s_k[0][0])[i] = v4u{0, 0, 0, 0};
      reinterpret_cast<v4u*>(&s_v[0][0])[i] = v4u{0, 0, 0, 0};
    }
    __syncthreads();
  }

  const int wr = wave * 16 * RT;  // the wave's first row of the tile
  const int wrows = min(max(it.count - wr, 0), 16 * RT);
  int row[RT], lim[RT];
  bool valid[RT];
  float c[RT], m[RT], l[RT];
  v4u q[RT][NP][DP / 32];
  v4f o[RT][NC];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    valid[t] = 16 * t + n < wrows;
    row[t] = it.first + (valid[t] ? wr + 16 * t + n : 0);
    const int token = row[t] / a.group;
    lim[t] = valid[t] ? own_limit(a, it, token) : 0;
    c[t] = load_q<T, TC, DP>(a, valid[t], token, it.head * a.group + row[t] % a.group, g, q[t]);
    m[t] = -INFINITY;
    l[t] = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) o[t][i] = v4f{0, 0, 0, 0};
  }
  // own keys that the wave's first and last row see
  const int least = wrows > 0 ? own_limit(a, it, (it.first + wr) / a.group) : 0;
  const int most = wrows > 0 ? own_limit(a, it, (it.first + wr + wrows - 1) / a.group) : 0;
  bool bad = false;

  const CacheArgs& ca = a.cache;
  const int32_t* own_pages = a.pages + (int64_t)max(it.b, 0) * a.pages_stride;
  const int tiles_p = (it.pk1 - it.pk0 + KT - 1) / KT;
  const int tiles = tiles_p + max(0, (it.ok1 - it.ok0 + KT - 1) / KT);

  auto issue = [&](int tile, int buf) {
    const bool pre = tile < tiles_p;
    const int32_t* pages = pre ? a.prefix_pages : own_pages;
    const int kend = pre ? it.pk1 : it.ok1;
    const int kb = (pre ? it.pk0 + tile * KT : it.ok0 + (tile - tiles_p) * KT) + wave * KW;
    const int in = min(kb, kend - 1);
    const int p = in / ca.page_size;
    int id = uniform(pages[p]);
    if ((u32)id >= (u32)ca.n_pages) {
      bad = true;
      id = 0;
    }
    const int64_t base = (int64_t)id * ca.page + (int64_t)it.head * ca.head;
    const uint16_t *kp = ca.k + base, *vp = ca.v + base;
    const int start = p * ca.page_size;
#pragma unroll
    for (int i = 0; i < KW / KI; ++i) {
      const int local = wave * KW + i * KI + lane / CH, pos = lane % CH;
      const int64_t at = (int64_t)(min(kb + i * KI + lane / CH, kend - 1) - start) * ca.token;
      const int ck = pos ^ swizzle_k<DP>(local), cv = pos ^ swizzle_v<DP>(local);
      if (ck * 8 < a.dim)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kp + at + ck * 8),
                                         (DQ_LDS(void)*)&s_k[buf][(wave * KW + i * KI) * DP], 16, 0, 0);
      if (cv * 8 < a.dim)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vp + at + cv * 8),
                                         (DQ_LDS(void)*)&s_v[buf][(wave * KW + i * KI) * DP], 16, 0, 0);
    }
  };

  auto compute = [&](int kb, const int (&limit)[RT], int least_, int most_, const uint16_t* sk, const uint16_t* sv) {
    if (kb >= most_) return;
    v4f s[RT][KT / 16];
#pragma unroll
    for (int u = 0; u < KT / 16; ++u) {
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t][u] = v4f{0, 0, 0, 0};
      const int key = 16 * u + n;
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) {
        const v4u kf = *reinterpret_cast<const v4u*>(sk + key * DP + ((4 * e + g) ^ swizzle_k<DP>(key)) * 8);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) s[t][u] = mma<TC>(kf, q[t][p][e], s[t][u]);
      }
    }
    const bool edge = kb + KT > least_;
    u32 pw[RT][NP][KT / 32][4];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float x[KT / 4];
#pragma unroll
      for (int u = 0; u < KT / 16; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[4 * u + i] = s[t][u][i];
          if (edge) x[4 * u + i] = kb + 16 * u + 4 * g + i < limit[t] ? x[4 * u + i] : -INFINITY;
        }
      const float alpha = softmax_step<TC, KT / 4>(x, c[t], m[t], l[t]);
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int i = 0; i < NC; ++i) o[t][i] *= alpha;
      }
#pragma unroll
      for (int u = 0; u < KT / 8; ++u) {
        u32 parts[NP];
        split<T, TC>(x[2 * u], x[2 * u + 1], parts);
#pragma unroll
        for (int p = 0; p < NP; ++p) pw[t][p][u / 4][u % 4] = parts[p];
      }
    }
    auto value = [&](int u, int i) {  // the operand of values 16 i .. + 15 and keys 32 u .. + 31
      v4u x;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = 32 * u + 16 * h + 4 * g + (n >> 2);
        const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (DQ_LDS(v4s)*)(sv + key * DP + ((2 * i + ((n >> 1) & 1)) ^ swizzle_v<DP>(key)) * 8 + (n & 1) * 4));
        const v2u z = __builtin_bit_cast(v2u, y);
        x[2 * h] = z[0];
        x[2 * h + 1] = z[1];
      }
      return x;
    };
    if (!edge) {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const v4u vt = value(u, i);
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
              o[t][i] = mma<TC>(vt, v4u{pw[t][p][u][0], pw[t][p][u][1], pw[t][p][u][2], pw[t][p][u][3]}, o[t][i]);
        }
    } else {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) {
        v4u sees[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + 32 * u + 16 * (j >> 1) + 4 * g + 2 * (j & 1);
            sees[t][j] = (key < limit[t] ? kOne<TC> : 0u) | (key + 1 < limit[t] ? kOne<TC> << 16 : 0u);
          }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          v4u vt = value(u, i);
          if (__any(has_nonfinite<TC>(vt))) {
            v4u pos, neg;
            take_nonfinite<TC>(vt, pos, neg);
#pragma unroll
            for (int t = 0; t < RT; ++t) o[t][i] = add_nonfinite<TC>(pos, neg, sees[t], o[t][i]);
          }
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
              o[t][i] = mma<TC>(vt, v4u{pw[t][p][u][0], pw[t][p][u][1], pw[t][p][u][2], pw[t][p][u][3]}, o[t][i]);
        }
      }
    }
  };

  int pre_lim[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) pre_lim[t] = valid[t] ? it.pk1 : 0;
  const int pre = wrows > 0 ? it.pk1 : 0;
  if (tiles > 0) issue(0, 0);
  for (int tile = 0; tile < tiles; ++tile) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile is in LDS
    __syncthreads();                     // everyone's is, and the other buffer is read out
    if (tile + 1 < tiles) issue(tile + 1, (tile + 1) & 1);
    const uint16_t *sk = s_k[tile & 1], *sv = s_v[tile & 1];
    if (tile < tiles_p)
      compute(it.pk0 + tile * KT, pre_lim, pre, pre, sk, sv);
    else
      compute(it.ok0 + (tile - tiles_p) * KT, lim, least, most, sk, sv);
  }
  if (bad) s_bad = 1;
  __syncthreads();
  const bool nan = s_bad != 0;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float sum = row_sum(l[t]);
    if (nan) sum = __builtin_nanf("");
    if (!valid[t]) continue;
    const int tk = row[t] / a.group, h = it.head * a.group + row[t] % a.group;
    if (a.part_o == nullptr) {
      if (it.b < 0 && a.q_offsets != nullptr && (tk < a.q_offsets[0] || tk >= a.q_offsets[a.batch])) continue;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at = (int64_t)tk * a.out_token + (int64_t)h * a.out_head;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (16 * i + 4 * g < a.dim) store4<T>(a, at, 16 * i + 4 * g, o[t][i] * inv);
      if (a.lse != nullptr && g == 0) a.lse[(int64_t)tk * a.heads + h] = lse_of(m[t], sum, kShift<TC>);
    } else {
      const int64_t at = ((int64_t)it.slot * ca.kv_heads + it.head) * a.tokens * a.group + row[t];
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (16 * i + 4 * g < a.dim) *reinterpret_cast<v4f*>(a.part_o + at * a.dim + 16 * i + 4 * g) = o[t][i];
      if (g == 0) *reinterpret_cast<v2f*>(a.part_ml + at * 2) = v2f{m[t], sum};
    }
  }
}

// ---- the join: the parts of a row, one wave a row ----------------------------

// The sequence of token t: the last b with q_offsets[b] <= t (-1: none).
DQ_DEV int find_seq(const AttnArgs& a, int t) {
  if (a.q_offsets == nullptr) return t;
  int lo = -1, hi = a.batch;  // q_offsets[lo] <= t < q_offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.q_offsets[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo >= 0 && t < a.q_offsets[lo + 1] ? lo : -1;
}

template <int T, int TC>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, AttnPart wa, AttnPart wb) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  const int t = uniform((int)(id / a.heads)), h = uniform((int)(id % a.heads));
  if (t >= a.tokens) return;
  const int b = find_seq(a, t);
  if (b < 0) return;
  // the own parts that were written: those that begin inside the sequence, and the first
  const int len = a.max_len > 0 ? min(max(a.lens[b], 0), a.max_len) : 0;
  const int end = wb.with_prefix ? (len > 0 ? wb.own_from + len : a.prefix_len) : len;
  const int own = min(wb.splits, max(1, (end + wb.chunk - 1) / max(wb.chunk, 1)));
  const int parts = wa.splits + (wb.splits > 0 ? own : 0);
  const int64_t R = (int64_t)a.tokens * a.group, step = R * a.cache.kv_heads;
  const int64_t at = (int64_t)(h / a.group) * R + (int64_t)t * a.group + h % a.group;
  float mx = -INFINITY;
  for (int s = lane; s < parts; s += 64) mx = fmaxf(mx, a.part_ml[(at + s * step) * 2]);
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
  const float base = mx == -INFINITY ? 0.f : mx;
  v4f y = {0, 0, 0, 0};
  float sum = 0;
  const int d = 4 * lane;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const v2f ml = *reinterpret_cast<const v2f*>(a.part_ml + (at + s * step) * 2);
    const float f = exp2_fast(ml[0] - base);
    sum = fmaf(ml[1], f, sum);
    if (d < a.dim) {
      const v4f x = *reinterpret_cast<const v4f*>(a.part_o + (at + s * step) * a.dim + d);
      y += f > 0.f ? x * f : v4f{0, 0, 0, 0};
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (d < a.dim) store4<T>(a, (int64_t)t * a.out_token + (int64_t)h * a.out_head, d, y * inv);
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)t * a.heads + h] = lse_of(mx, sum, kShift<TC>);
}

template <int T, int TC, int DP>
hipError_t launch_part(const AttnArgs& a, const AttnPart& w, bool stacked, hipStream_t s) {
  const uint32_t items = (uint32_t)((int64_t)w.tiles * a.cache.kv_heads * w.splits * (stacked ? 1 : a.batch));
  if (w.rows == 16)
    hipLaunchKernelGGL((k_attn_few<T, TC, DP>), dim3(items), dim3(256), 0, s, a, w, stacked);
  else if (w.rows == 64)
    hipLaunchKernelGGL((k_attn_tile<T, TC, DP, 1>), dim3(items), dim3(256), 0, s, a, w, stacked);
  else if constexpr (T != DQ_F32)
    hipLaunchKernelGGL((k_attn_tile<T, TC, DP, 2>), dim3(items), dim3(256), 0, s, a, w, stacked);
  return hipGetLastError();
}

template <int T, int TC, int DP>
hipError_t launch(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  if (p.shared.splits > 0)
    if (hipError_t e = launch_part<T, TC, DP>(a, p.shared, true, s); e != hipSuccess) return e;
  if (p.own.splits > 0)
    if (hipError_t e = launch_part<T, TC, DP>(a, p.own, false, s); e != hipSuccess) return e;
  if (a.part_o == nullptr) return hipSuccess;
  hipLaunchKernelGGL((k_attn_join<T, TC>), dim3((uint32_t)(((int64_t)a.tokens * a.heads + 3) / 4)), dim3(256), 0, s, a, p.shared,
                     p.own);
  return hipGetLastError();
}

template <int T, int TC>
hipError_t by_dim(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  if (a.dim <= 64) return launch<T, TC, 64>(a, p, s);
  if (a.dim <= 128) return launch<T, TC, 128>(a, p, s);
  return launch<T, TC, 256>(a, p, s);
}

}  // namespace

hipError_t launch_attention(int type, int cache_type, const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  if (cache_type == DQ_F16) return type == DQ_F32 ? by_dim<DQ_F32, DQ_F16>(a, p, s) : by_dim<DQ_F16, DQ_F16>(a, p, s);
  return type == DQ_F32 ? by_dim<DQ_F32, DQ_BF16>(a, p, s) : by_dim<DQ_BF16, DQ_BF16>(a, p, s);
}

}  // namespace dq
