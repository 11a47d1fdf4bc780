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
//
// What bounds it (bf16, head size 128; a copy of 1 GiB reaches 4.8 TB/s here, a matrix product of 8,192^3
// 1,150 to 1,190 TFLOP/s): the bytes of the keys and values where rows are few, the matrix cores and the vector
// unit, which share their issue slots, where they are many; the launch and one chain of dependent reads (offsets,
// page numbers, keys: 7 us) where both are few.
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
typedef unsigned short v2us __attribute__((ext_vector_type(2)));

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

// A load of 16 bytes a lane straight to LDS: lane l's from base + off to the LDS address lds + 16 l. Written
// as an instruction because the compiler would wait for every load under way before any read of
// LDS; the wait is where the tile changes hands (wait_loads, then the barrier). M0, which holds the
// LDS address, is left as it was.
DQ_DEV void load_to_lds(const void* base, u32 off, u32 lds) {
  u32 m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
      : "=&s"(m0)
      : "s"(lds), "v"(off), "s"(base)
      : "memory");
}
// The same for N rows of 1,024 bytes of LDS in one go: load i is offset by 1,024 i on both sides (off[i] leaves
// that out).
template <int N>
DQ_DEV void load_rows_to_lds(const void* base, const u32 (&off)[N], u32 lds) {
  static_assert(N == 2 || N == 4);
  u32 m0;
  if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\t"
        "global_load_lds_dwordx4 %3, %4 offset:1024\n\ts_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(lds), "v"(off[0]), "v"(off[1]), "s"(base)
        : "memory");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %6\n\t"
        "global_load_lds_dwordx4 %3, %6 offset:1024\n\tglobal_load_lds_dwordx4 %4, %6 offset:2048\n\t"
        "global_load_lds_dwordx4 %5, %6 offset:3072\n\ts_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base)
        : "memory");
}
// The same where rows may be less than 1,024 bytes apart: off[i] is the whole offset.
template <int N>
DQ_DEV void load_near_rows_to_lds(const void* base, const u32 (&off)[N], u32 lds) {
  static_assert(N == 2 || N == 4);
  u32 m0;
  if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %4\n\ts_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(lds), "v"(off[0]), "v"(off[1]), "s"(base)
        : "memory", "scc");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %6\n\ts_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(lds), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base)
        : "memory", "scc");
}
DQ_DEV void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}
DQ_DEV u32 lds_address(const void* p) { return (u32)(uintptr_t)(DQ_LDS(const void)*)p; }

// A page number through the scalar cache.
DQ_DEV int page_at(const int32_t* pages, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)pages)[i];
}

// Where a run of keys lies in its pages: key `key` is place `in` of entry `p` of the page list.
struct PageWalk {
  int key, p, in;
  DQ_DEV void start(int k, int page_size) {
    key = k;
    p = k / page_size;
    in = k - p * page_size;
  }
  // `pages` whole pages and `rest` places on
  DQ_DEV void skip(int keys, int pages, int rest, int page_size) {
    key += keys;
    p += pages;
    in += rest;
    if (in >= page_size) {
      in -= page_size;
      ++p;
    }
  }
};

// ---- infinite and NaN values that only some rows of a tile see ------------
// A masked key has weight 0, but 0 times an infinite value is NaN in a matrix product. In tiles
// that some rows see in part, such values are taken out of the product and noted, and the rows that
// see them get them at the end. A row sees every key that an earlier row of its item sees, so
// the first row is all that is noted of a value's column: first[0] for +inf and NaN, first[1]
// for -inf and NaN.
template <int TC>
constexpr u32 kExp = TC == DQ_F16 ? 0x7C00u : 0x7F80u;

template <int TC>
DQ_DEV bool nonfinite(u32 x) {
  return (x & kExp<TC>) == kExp<TC> || (x & (kExp<TC> << 16)) == (kExp<TC> << 16);
}
// Notes the infinite and NaN values of a dword (columns d, d + 1; seen from row `row` on, by none if
// it is past the item) and returns it without them.
template <int TC, int DP>
DQ_DEV u32 take_nonfinite(u32 x, int d, int row, int rows, int (&first)[2][DP]) {
  u32 clean = 0;
  for (int h = 0; h < 2; ++h) {
    const u32 v = (x >> (16 * h)) & 0xFFFFu;
    if ((v & kExp<TC>) != kExp<TC>) {
      clean |= v << (16 * h);
    } else if (row < rows) {
      const bool nan = (v & 0x7FFFu) != kExp<TC>;
      if (nan || v < 0x8000u) atomicMin(&first[0][d + h], row);
      if (nan || v >= 0x8000u) atomicMin(&first[1][d + h], row);
    }
  }
  return clean;
}
template <int DP>
DQ_DEV float noted(const int (&first)[2][DP], int row, int d) {
  return (row >= first[0][d] ? INFINITY : 0.f) + (row >= first[1][d] ? -INFINITY : 0.f);
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
  int part0;         // the row that the workspace's parts begin with
};

// The first token of a launch's sequences.
DQ_DEV int first_token(const AttnArgs& a) { return a.sliced ? min(max(a.q_offsets[0], 0), a.tokens) : 0; }

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
  const int t0 = first_token(a), end = t0 + min(a.part_tokens, a.tokens - t0);
  it.part0 = t0 * a.group;
  it.pk0 = it.pk1 = it.ok0 = it.ok1 = 0;
  if (stacked) {
    it.b = -1;
    it.count = min(tile, (end - t0) * a.group - t * tile);
    if (it.count <= 0) return false;
    it.first = t0 * a.group + t * tile;
    it.token0 = it.own0 = it.len = 0;
    it.pk0 = k0;
    it.pk1 = min(k1, a.prefix_len);
    return true;
  }
  const int b = rest / w.splits;
  it.b = b;
  const int lo = a.q_offsets != nullptr ? a.q_offsets[b] : b;
  const int hi = a.q_offsets != nullptr ? a.q_offsets[b + 1] : b + 1;
  const int len = a.max_len > 0 ? a.lens[b] : 0;  // (all three under way together)
  // (whatever the offsets hold, rows stay inside the tensors)
  const int first = min(max(lo, t0), end);
  const int n = min(min(max(hi, first), end) - first, a.max_q);
  const int tt = w.backward ? w.tiles - 1 - t : t;
  it.count = min(tile, n * a.group - tt * tile);
  if (it.count <= 0) return false;
  it.first = first * a.group + tt * tile;
  it.len = min(max(len, 0), a.max_len);
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

// The first row of the item that sees own key `key` (its count or more: none does); of the
// prefix every row sees every key.
DQ_DEV int first_row(const AttnArgs& a, const Item& it, int key) {
  return max(0, (it.token0 + key + 1 - it.own0) * a.group - it.first);
}

// The query fragments of rows: lane l has row l % 16 and, of every 32 values, 8 (l / 16) .. + 7. First their loads,
// then, once other loads are under way too, the operands; the latter returns
// the factor from products to scores in powers of two: fp32 rows are scaled to a largest value
// in [2^14, 2^15), where all of their parts are normal numbers.
template <int T, int DP>
struct RawQ {
  v4u x[DP / 32][T == DQ_F32 ? 2 : 1];
};
template <int T, int DP>
DQ_DEV void load_q(const AttnArgs& a, bool valid, int token, int head, int g, RawQ<T, DP>& r) {
  const int64_t base = (int64_t)token * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) {
    const int d = 32 * s + 8 * g;
#pragma unroll
    for (int k = 0; k < (T == DQ_F32 ? 2 : 1); ++k) {
      v4u x = {0, 0, 0, 0};
      if (valid && d < a.dim) {
        if constexpr (T == DQ_F32) {
          const float* p = static_cast<const float*>(a.q) + base + d + 4 * k;
          if (a.q_vec)
            x = *reinterpret_cast<const v4u*>(p);
          else
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = as_u(p[i]);
        } else {
          const uint16_t* p = static_cast<const uint16_t*>(a.q) + base + d;
          if (a.q_vec)
            x = *reinterpret_cast<const v4u*>(p);
          else
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (u32)p[2 * i] | ((u32)p[2 * i + 1] << 16);
        }
      }
      r.x[s][k] = x;
    }
  }
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

// ---- few rows: up to 16 of one item ----------------------------------------
// The four waves take 32 keys each in turn, with a running softmax of their own, and add up at
// the end: a decode step's own keys, where a tile of 16 rows is mostly empty and the keys' bytes
// are all that counts. Keys and values go straight from memory to registers: a lane's 16 bytes of a key
// are its A operand as they lie; of the values it takes DP / 16 of 8 keys, which v_perm turns into
// the operands of DP / 16 tiles. Bound by the reads: 128 sequences of up to 2,048 own keys, 4 kv heads of 128
// (403 MB), 81 us, 4.95 TB/s; 64 of up to 512, 8 kv heads (100 MB), 22 us; a tile of 64 rows in their place
// 50.7 us against 46.5 for 64 such sequences behind 8,192 shared keys.

template <int DP>
struct KvRegs {
  v4u k[2][DP / 32];
  u32 v[8][DP / 32];  // [key slot][dword]: DP / 16 values
};

template <int DP>
struct FewLds {
  v4f o[4][16][DP / 4];
  float ml[4][16][2];
  int first[2][DP];
  int bad, noted;
};

template <int T, int TC, int DP>
DQ_DEV void few_rows(const AttnArgs& a, const AttnPart& w, bool stacked, int index, FewLds<DP>& sh) {
  constexpr int NP = kParts<T, TC>;
  constexpr int NC = DP / 16;
  auto &s_o = sh.o;
  auto &s_ml = sh.ml;
  auto &s_first = sh.first;
  int &s_bad = sh.bad, &s_noted = sh.noted;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  Item it;
  if (!find_item(a, w, stacked, index, 16, it)) return;
  if (threadIdx.x == 0) s_bad = s_noted = 0;
  for (int i = threadIdx.x; i < 2 * DP; i += 256) (&s_first[0][0])[i] = 1 << 30;
  __syncthreads();

  const bool valid = n < it.count;
  const int row = it.first + (valid ? n : 0);
  const int token = row / a.group, qh = it.head * a.group + row % a.group;
  const int own_lim = own_limit(a, it, token);
  const int own_least = own_limit(a, it, it.first / a.group);
  RawQ<T, DP> raw;
  load_q<T, DP>(a, valid, token, qh, g, raw);
  v4u q[NP][DP / 32];
  float c = 1.f;

  RowMax rm;
  float l = 0;
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

  // The keys in tiles of 32, the prefix's before the own; a wave takes every fourth. The page numbers
  // of a tile are read one step ahead of its loads.
  const int tiles_p = (it.pk1 - it.pk0 + 31) / 32;
  const int tiles = tiles_p + max(0, (it.ok1 - it.ok0 + 31) / 32);
  const int32_t* own_pages = a.pages + (int64_t)max(it.b, 0) * a.pages_stride;
  struct Place {
    int id[2], in[2];  // of each half's page: its number, the half's first place
  };
  PageWalk walk;
  walk.key = -1;
  bool walk_pre = true;
  const int skip_pages = 128 / ca.page_size, skip_rest = 128 % ca.page_size;
  auto place = [&](int tile) {  // tiles wave, wave + 4, ... in turn
    const bool pre = tile < tiles_p;
    const int32_t* pages = pre ? a.prefix_pages : own_pages;
    if (walk.key < 0 || walk_pre != pre)
      walk.start(pre ? it.pk0 + tile * 32 : it.ok0 + (tile - tiles_p) * 32, ca.page_size);
    else
      walk.skip(128, skip_pages, skip_rest, ca.page_size);
    walk_pre = pre;
    Place r;
    r.id[0] = r.id[1] = page_at(pages, walk.p);
    r.in[0] = r.in[1] = walk.in;
    if (walk.key + 16 < (pre ? it.pk1 : it.ok1)) {  // (else the second half's keys do not count)
      const bool over = walk.in + 16 == ca.page_size;
      if (over) r.id[1] = page_at(pages, walk.p + 1);
      r.in[1] = over ? 0 : walk.in + 16;
    }
    return r;
  };
  auto load = [&](const Place& pl, KvRegs<DP>& r) {
    int64_t base[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int id = pl.id[t];
      if ((u32)id >= (u32)ca.n_pages) {
        bad = true;
        id = 0;
      }
      base[t] = (int64_t)id * ca.page + (int64_t)pl.in[t] * ca.token + (int64_t)it.head * ca.head;
    }
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
  auto compute = [&](int tile, KvRegs<DP>& r) {
    const bool own = tile >= tiles_p;
    const int kb = own ? it.ok0 + (tile - tiles_p) * 32 : it.pk0 + tile * 32;
    const int kend = own ? it.ok1 : it.pk1;
    const int lim = !valid ? 0 : own ? own_lim : it.pk1, least = own ? own_least : it.pk1;
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
    if (kb + 32 > least || kb + 32 > kend) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
        x[j] = key < lim && key < kend ? x[j] : -INFINITY;
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
          if (key >= kend) r.v[j][e] = 0;  // places past the keys may hold anything
      }
    }
    if (kb + 32 > least && least < kend) {  // some row does not see all of the tile's keys
      v2us top = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(v2us, r.v[j][e] & 0x7FFF7FFFu));
      if (__any(top[0] >= kExp<TC> || top[1] >= kExp<TC>)) {
        if (lane == 0) s_noted = 1;
        u32* tmp = reinterpret_cast<u32*>(&s_o[wave][0][0]) + lane;
#pragma unroll
        for (int j = 0; j < 8 * (DP / 32); ++j) tmp[64 * j] = r.v[j / (DP / 32)][j % (DP / 32)];
#pragma unroll 1
        for (int j = 0; j < 8 * (DP / 32); ++j) {
          const int slot = j / (DP / 32), key = kb + 16 * (slot >> 2) + 4 * g + (slot & 3);
          if (nonfinite<TC>(tmp[64 * j]))
            tmp[64 * j] = take_nonfinite<TC, DP>(tmp[64 * j], n * NC + j % (DP / 32) * 2, own ? first_row(a, it, key) : 0,
                                                 it.count, s_first);
        }
#pragma unroll
        for (int j = 0; j < 8 * (DP / 32); ++j) r.v[j / (DP / 32)][j % (DP / 32)] = tmp[64 * j];
      }
    }
    float mx;
    if (__any(passes<8>(x, c, rm, mx))) {
      const float alpha = move_max<TC>(mx, c, rm);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NC; ++i) o[i] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = exp2_fast(fmaf(x[j], c, -rm.base));
      l += x[j];
    }
    v4u p[NP];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32 parts[NP];
      split<T, TC>(x[2 * j], x[2 * j + 1], parts);
#pragma unroll
      for (int k = 0; k < NP; ++k) p[k][j] = parts[k];
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      v4u vt;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vt[e] = __builtin_amdgcn_perm(r.v[2 * e + 1][i >> 1], r.v[2 * e][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int k = NP - 1; k >= 0; --k) o[i] = mma<TC>(vt, p[k], o[i]);
    }
  };
  // (One tile's registers: two, one loading while the other is used, measured the same.)
  int tile = wave;
  Place next;
  KvRegs<DP> r;
  if (tile < tiles) {
    load(place(tile), r);
    if (tile + 4 < tiles) next = place(tile + 4);
  }
  c = q_operands<T, TC, DP>(a, raw, q);
  while (tile < tiles) {
    compute(tile, r);
    tile += 4;
    if (tile < tiles) {
      load(next, r);
      if (tile + 4 < tiles) next = place(tile + 4);
    }
  }

  // the waves' sums join in LDS
  l = row_sum(l);
  if (g == 0) {
    s_ml[wave][n][0] = rm.m;
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
      y += s_o[k][r][d4] * f;
    }
    if (s_bad) sum = __builtin_nanf("");
    if (s_noted)
      for (int e = 0; e < 4; ++e) y[e] += noted<DP>(s_first, r, 4 * d4 + e);
    const int rw = it.first + r, tk = rw / a.group, h = it.head * a.group + rw % a.group;
    if (a.part_o == nullptr) {
      if (it.b < 0 && a.q_offsets != nullptr && (tk < a.q_offsets[0] || tk >= a.q_offsets[a.batch])) continue;
      store4<T>(a, (int64_t)tk * a.out_token + (int64_t)h * a.out_head, 4 * d4, finish(y, sum, 1.f / sum));
      if (a.lse != nullptr && d4 == 0) a.lse[(int64_t)tk * a.heads + h] = lse_of(mx, sum, kShift<TC>);
    } else {
      const int64_t at = ((int64_t)it.slot * ca.kv_heads + it.head) * a.part_tokens * a.group + rw - it.part0;
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
//
// 8 sequences of 257 to 512 new tokens behind 8,192 shared keys, 32 / 8 bf16 heads of 128 (432 GFLOP): 495 to 525 us, 820 to 870
// TFLOP/s; a prompt of 4,096 in f16 (137 GFLOP, half of the square): 141 to 150 us, 915 to 970. Per wave and tile of 64 keys 64
// MFMAs (1,024 clocks at their rate) stand beside some 180 vector instructions, 32 of them exponentials:
// the matrix cores are busy 51% of the time, LDS 26% (no bank conflicts). Timing copies that leave a part out, of
// 527 us: the loads 65, the exponentials, their sums and rounding 70, the maxima 21, the reads of LDS 50; MFMAs alone
// 318. Measured and dropped: weights and scores of one tile in turn (555), tiles of 32 keys (605), 64
// rows a wave with one wave a SIMD (1,028), lines brought into the L2 four tiles ahead (627), maxima looked at
// after the weights (531).

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

template <int DP>
struct TileLds {
  uint16_t k[2][kTileKeys<DP> * DP];
  uint16_t v[2][kTileKeys<DP> * DP];
  int first[2][DP];
  int bad;
};

// DP: the values of a key's place in LDS, DC: those that the products run over (the head size, to the next 64, 96, 128, 192
// or 256).
template <int T, int TC, int DP, int DC, int RT>
DQ_DEV void many_rows(const AttnArgs& a, const AttnPart& w, bool stacked, int index, TileLds<DP>& sh) {
  constexpr int NP = kParts<T, TC>;
  constexpr int NC = DC / 16, KT = kTileKeys<DP>, CH = DP / 8;
  constexpr int KW = KT / 4, KI = 64 / CH;  // keys a wave loads of a tile, and with one instruction
  auto &s_k = sh.k, &s_v = sh.v;
  auto& s_first = sh.first;
  int& s_bad = sh.bad;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  Item it;
  if (!find_item(a, w, stacked, index, 64 * RT, it)) return;
  if (threadIdx.x == 0) s_bad = 0;
  for (int i = threadIdx.x; i < 2 * DP; i += 256) (&s_first[0][0])[i] = 1 << 30;
  if (a.dim < DP) {  // the loads leave the places past a head's values as they are: zero
    for (int i = threadIdx.x; i < 2 * KT * DP / 8; i += 256) {
      reinterpret_cast<v4u*>(&s_k[0][0])[i] = v4u{0, 0, 0, 0};
      reinterpret_cast<v4u*>(&s_v[0][0])[i] = v4u{0, 0, 0, 0};
    }
    __syncthreads();
  }

  const int wr = wave * 16 * RT;  // the wave's first row of the tile
  const int wrows = min(max(it.count - wr, 0), 16 * RT);
  int own_lim[RT];
  float c[RT];
  RowMax rm[RT];
  float l[RT];
  RawQ<T, DC> raw[RT];
  v4u q[RT][NP][DC / 32];
  v4f o[RT][NC];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const bool valid = 16 * t + n < wrows;
    const int row = it.first + (valid ? wr + 16 * t + n : 0);
    const int token = row / a.group;
    own_lim[t] = valid ? own_limit(a, it, token) : 0;
    load_q<T, DC>(a, valid, token, it.head * a.group + row % a.group, g, raw[t]);
    l[t] = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) o[t][i] = v4f{0, 0, 0, 0};
  }
  // own keys that the wave's first and last row see, and the item's first
  const int own_least = wrows > 0 ? own_limit(a, it, (it.first + wr) / a.group) : 0;
  const int item_least = own_limit(a, it, it.first / a.group);
  bool bad = false, noting = false;

  const CacheArgs& ca = a.cache;
  const u32 token_bytes = (u32)ca.token * 2;
  const int32_t* own_pages = a.pages + (int64_t)max(it.b, 0) * a.pages_stride;
  const int tiles_p = (it.pk1 - it.pk0 + KT - 1) / KT;
  const int tiles = tiles_p + max(0, (it.ok1 - it.ok0 + KT - 1) / KT);

  // This lane's loads of a whole tile and its reads (swizzle_k and swizzle_v repeat every 16 keys).
  const int lrow = lane / CH;
  auto kpos = [&](int i) { return (u32)((lane % CH) ^ swizzle_k<DP>(wave * KW + i * KI + lrow)) * 16; };
  auto vpos = [&](int i) { return (u32)((lane % CH) ^ swizzle_v<DP>(wave * KW + i * KI + lrow)) * 16; };
  u32 kload[KW / KI], vload[KW / KI];
#pragma unroll
  for (int i = 0; i < KW / KI; ++i) {
    // Heads of DP values lie 1,024 bytes apart from load to load at least. Places past a head of DC < DP values are not
    // read: the first chunk fills them.
    const u32 k = kpos(i), v = vpos(i), less = DC == DP ? 1024 * i : 0;
    kload[i] = (i * KI + lrow) * token_bytes + (k < DC * 2 ? k : 0) - less;
    vload[i] = (i * KI + lrow) * token_bytes + (v < DC * 2 ? v : 0) - less;
  }
  u32 kread[DC / 32], vread[NC];
#pragma unroll
  for (int e = 0; e < DC / 32; ++e) kread[e] = n * DP + ((4 * e + g) ^ swizzle_k<DP>(n)) * 8;
  const int vkey = 4 * g + (n >> 2);
#pragma unroll
  for (int i = 0; i < NC; ++i) vread[i] = vkey * DP + ((2 * i + ((n >> 1) & 1)) ^ swizzle_v<DP>(vkey)) * 8 + (n & 1) * 4;

  // The wave's keys of a tile lie in one page; its number is read one tile ahead of the loads.
  struct Place {
    int id, in, last;  // the page, the wave's first place of it, and the last place that counts after that
  };
  PageWalk walk;
  walk.key = -1;
  bool walk_pre = true;
  const int skip_pages = KT / ca.page_size, skip_rest = KT % ca.page_size;
  auto place = [&](int tile) {  // the tiles in turn
    const bool pre = tile < tiles_p;
    const int32_t* pages = pre ? a.prefix_pages : own_pages;
    const int kend = pre ? it.pk1 : it.ok1;
    if (walk.key < 0 || walk_pre != pre)
      walk.start((pre ? it.pk0 + tile * KT : it.ok0 + (tile - tiles_p) * KT) + wave * KW, ca.page_size);
    else
      walk.skip(KT, skip_pages, skip_rest, ca.page_size);
    walk_pre = pre;
    PageWalk at = walk;
    if (at.key >= kend) at.start(kend - 1, ca.page_size);  // past the keys the last one is loaded again
    return Place{page_at(pages, at.p), at.in, kend - 1 - at.key};
  };
  const u32 lds_k = lds_address(&s_k[0][wave * KW * DP]), lds_v = lds_address(&s_v[0][wave * KW * DP]);
  struct Source {
    int64_t base;  // of the wave's first key
    int last;
  };
  const int64_t head_at = (int64_t)it.head * ca.head;
  auto resolve = [&](const Place& r) {
    int id = r.id;
    if ((u32)id >= (u32)ca.n_pages) {
      bad = true;
      id = 0;
    }
    return Source{(int64_t)id * ca.page + (int64_t)r.in * ca.token + head_at, r.last};
  };
  auto issue = [&](const uint16_t* pool, const Source& r, const u32 (&off)[KW / KI], auto pos_of, u32 to) {
    const uint16_t* from = pool + r.base;
    if (r.last >= KW - 1 && a.dim == DC) {
      if constexpr (DC == DP)
        load_rows_to_lds(from, off, to);
      else
        load_near_rows_to_lds(from, off, to);
    } else {
#pragma unroll
      for (int i = 0; i < KW / KI; ++i) {
        const u32 at = (u32)min(i * KI + lrow, r.last) * token_bytes, pos = pos_of(i);
        if (pos < (u32)a.dim * 2) load_to_lds(from, at + pos, to + i * 1024);
      }
    }
  };
  auto issue_keys = [&](const Source& r, int buf) { issue(ca.k, r, kload, kpos, lds_k + buf * KT * DP * 2); };
  auto issue_values = [&](const Source& r, int buf) { issue(ca.v, r, vload, vpos, lds_v + buf * KT * DP * 2); };
  auto first_key = [&](int tile) { return tile < tiles_p ? it.pk0 + tile * KT : it.ok0 + (tile - tiles_p) * KT; };

  // S^T of a tile
  auto scores = [&](const uint16_t* sk, v4f (&s)[RT][KT / 16]) {
#pragma unroll
    for (int e = 0; e < DC / 32; ++e)
#pragma unroll
      for (int u = 0; u < KT / 16; ++u) {
        const v4u kf = *reinterpret_cast<const v4u*>(sk + kread[e] + 16 * u * DP);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if (e == 0) s[t][u] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) s[t][u] = mma<TC>(kf, q[t][p][e], s[t][u]);
        }
      }
  };
  // One pair of weights of scores whose maxima have been looked at.
  auto weigh = [&](const v4f (&s)[RT][KT / 16], int pair, u32 (&pw)[RT][NP][KT / 32][4]) {
    const int t = pair / (KT / 8), u = pair % (KT / 8) / 2, i = pair % 2 * 2;
    const float x0 = exp2_fast(fmaf(s[t][u][i], c[t], -rm[t].base));
    const float x1 = exp2_fast(fmaf(s[t][u][i + 1], c[t], -rm[t].base));
    l[t] += x0;
    l[t] += x1;
    u32 parts[NP];
    split<T, TC>(x0, x1, parts);
#pragma unroll
    for (int p = 0; p < NP; ++p) pw[t][p][u / 2][u % 2 * 2 + i / 2] = parts[p];
  };
  auto key_operand = [&](const uint16_t* sk, int i) {
    return *reinterpret_cast<const v4u*>(sk + kread[i / (KT / 16)] + i % (KT / 16) * 16 * DP);
  };
  auto value_operand = [&](const uint16_t* sv, int i) {
    v4u x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v2u z = __builtin_bit_cast(
          v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((DQ_LDS(v4s)*)(sv + vread[i % NC] + (i / NC * 32 + 16 * h) * DP)));
      x[2 * h] = z[0];
      x[2 * h + 1] = z[1];
    }
    return x;
  };

  // Keys run one tile before values: while a tile's weights are computed, which is vector work,
  // the matrix cores form the next tile's scores.
  v4f s[RT][KT / 16];
  Source next = {};   // the next tile's
  Place after = {};   // and where the one after it lies
  if (tiles > 0) {
    const Place p0 = place(0);
    const Place p1 = tiles > 1 ? place(1) : p0;
    if (tiles > 2) after = place(2);
    const Source first = resolve(p0);
    next = resolve(p1);
    issue_keys(first, 0);
    issue_values(first, 0);
    if (tiles > 1) issue_keys(next, 1);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) c[t] = q_operands<T, TC, DC>(a, raw[t], q[t]);
  // (waits outside the branch, so that the compiler sees q's loads end here and adds no wait to the loop)
  wait_loads();
  __syncthreads();
  if (tiles > 0) scores(s_k[0], s);
  for (int tile = 0; tile < tiles; ++tile) {
    if (tile > 0) wait_loads();  // this wave's part of the tile's values and of the next one's keys is in LDS
    __syncthreads();             // everyone's is, and the buffers loaded below are read out (tile 0: its keys, just above)
    if (tile + 1 < tiles) issue_values(next, (tile + 1) & 1);
    if (tile + 2 < tiles) {
      next = resolve(after);
      issue_keys(next, tile & 1);
      if (tile + 3 < tiles) after = place(tile + 3);
    }
    const bool pre = tile < tiles_p;
    const int kb = first_key(tile);
    const int least = wrows == 0 ? 0 : pre ? it.pk1 : own_least;
    const uint16_t* sk = s_k[(tile + 1) & 1];
    uint16_t* sv = s_v[tile & 1];

    if (kb + KT > (pre ? it.pk1 : item_least)) {  // some row sees the tile in part
      bool nf = false;
      for (int i = threadIdx.x; i < KT * DP / 2; i += 256) nf |= nonfinite<TC>(reinterpret_cast<const u32*>(sv)[i]);
      if (__syncthreads_or(nf)) {
        noting = true;
        for (int i = threadIdx.x; i < KT * DP / 2; i += 256) {
          const u32 x = reinterpret_cast<const u32*>(sv)[i];
          if (!nonfinite<TC>(x)) continue;
          const int local = i / (DP / 2), pos = i % (DP / 2) / 4;
          const int d = (pos ^ swizzle_v<DP>(local)) * 8 + i % 4 * 2, key = kb + local;
          const int from = key >= (pre ? it.pk1 : it.ok1) ? it.count : pre ? 0 : first_row(a, it, key);
          reinterpret_cast<u32*>(sv)[i] = take_nonfinite<TC, DP>(x, d, from, it.count, s_first);
        }
        __syncthreads();
      }
    }
    if (kb + KT > least) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int lim = wrows == 0 ? 0 : pre ? it.pk1 : own_lim[t];
#pragma unroll
        for (int u = 0; u < KT / 16; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (kb + 16 * u + 4 * g + i >= lim) s[t][u][i] = -INFINITY;
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float x[KT / 4], mx;
#pragma unroll
      for (int i = 0; i < KT / 4; ++i) x[i] = s[t][i / 4][i % 4];
      if (__any(passes<KT / 4>(x, c[t], rm[t], mx))) {
        const float alpha = move_max<TC>(mx, c[t], rm[t]);
        l[t] *= alpha;
#pragma unroll
        for (int i = 0; i < NC; ++i) o[t][i] *= alpha;
      }
    }
    // The order below is kept (sched_barrier): operands are read kAhead steps before their products, and
    // the vector work of the weights goes between the products of the next tile's scores.
    constexpr int F = KT * DC / 512, kAhead = 4, kPairs = RT * KT / 8;
    u32 pw[RT][NP][KT / 32][4];
    v4f ahead[RT][KT / 16];  // (after the last tile of what the buffer holds: not used)
    v4u ring[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ring[i] = key_operand(sk, i);
    __builtin_amdgcn_s_setprio(1);  // (the other wave of the SIMD is then in its scalar and vector work)
#pragma unroll
    for (int i = 0; i < F; ++i) {
      const int e = i / (KT / 16), u = i % (KT / 16);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if (e == 0) ahead[t][u] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) ahead[t][u] = mma<TC>(ring[i % kAhead], q[t][p][e], ahead[t][u]);
      }
      ring[i % kAhead] = i + kAhead < F ? key_operand(sk, i + kAhead) : value_operand(sv, i + kAhead - F);
#pragma unroll
      for (int k = i * kPairs / F; k < (i + 1) * kPairs / F; ++k) weigh(s, k, pw);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < F; ++i) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {
          const u32(&w4)[4] = pw[t][p][i / NC];
          o[t][i % NC] = mma<TC>(ring[i % kAhead], v4u{w4[0], w4[1], w4[2], w4[3]}, o[t][i % NC]);
        }
      if (i + kAhead < F) ring[i % kAhead] = value_operand(sv, i + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int u = 0; u < KT / 16; ++u) s[t][u] = ahead[t][u];
  }
  if (bad) s_bad = 1;
  __syncthreads();
  const bool nan = s_bad != 0;
  float* s_sum = reinterpret_cast<float*>(&s_k[0][0]);  // (the keys have been read)
  const int64_t part = ((int64_t)it.slot * ca.kv_heads + it.head) * a.part_tokens * a.group - it.part0;
  auto covered = [&](int token) {
    return it.b >= 0 || a.q_offsets == nullptr || (token >= a.q_offsets[0] && token < a.q_offsets[a.batch]);
  };
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float sum = row_sum(l[t]);
    if (nan) sum = __builtin_nanf("");
    if (16 * t + n >= wrows) continue;
    const int row = it.first + wr + 16 * t + n, token = row / a.group, h = it.head * a.group + row % a.group;
    if (a.part_o == nullptr) {
      if (!covered(token)) continue;
      const float inv = 1.f / sum;
      const int64_t at = (int64_t)token * a.out_token + (int64_t)h * a.out_head;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (16 * i + 4 * g < a.dim) store4<T>(a, at, 16 * i + 4 * g, finish(o[t][i], sum, inv));
      if (a.lse != nullptr && g == 0) a.lse[(int64_t)token * a.heads + h] = lse_of(rm[t].m, sum, kShift<TC>);
      if (noting && g == 0) s_sum[wr + 16 * t + n] = sum;
    } else {
      const int64_t at = part + row;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (16 * i + 4 * g < a.dim) *reinterpret_cast<v4f*>(a.part_o + at * a.dim + 16 * i + 4 * g) = o[t][i];
      if (g == 0) *reinterpret_cast<v2f*>(a.part_ml + at * 2) = v2f{rm[t].m, sum};
    }
  }
  if (noting) {  // the infinite and NaN values go to what has just been written
    __syncthreads();
    for (int i = threadIdx.x; i < it.count * a.dim; i += 256) {
      const int r = i / a.dim, d = i % a.dim, row = it.first + r;
      const float y = noted<DP>(s_first, r, d);
      if (y == 0.f) continue;
      const int token = row / a.group;
      if (a.part_o != nullptr) {
        a.part_o[(part + row) * a.dim + d] += y;
      } else if (covered(token) && s_sum[r] != 0.f) {
        const int64_t at = (int64_t)token * a.out_token + (int64_t)(it.head * a.group + row % a.group) * a.out_head + d;
        store1<T>(a.out, at, load1<T>(a.out, at) + y);
      }
    }
  }
}

// ---- the launch: shared items, then own ones ---------------------------------

// Item of workgroup b of n. Workgroups go to the 8 XCDs in turn: consecutive items, which read the same keys for
// other rows, stay on one XCD and its L2.
DQ_DEV int xcd_item(int b, int n) {
  const int each = n / 8;
  return b < 8 * each ? b % 8 * each + b / 8 : b;
}

template <int T, int TC, int DP, int DC, int ROWS, class Lds>
DQ_DEV void run_item(const AttnArgs& a, const AttnPart& w, bool stacked, int index, Lds& sh) {
  if constexpr (ROWS == 16)
    few_rows<T, TC, DP>(a, w, stacked, index, sh.few);
  else
    many_rows<T, TC, DP, DC, ROWS / 64>(a, w, stacked, index, sh.tile);
}

template <int DP, int MOST>
union AttnLds {
  FewLds<DP> few;
  TileLds<DP> tile;
};
template <int DP>
union AttnLds<DP, 16> {
  FewLds<DP> few;
};

// Waves a SIMD that the registers are held down to. Two, but for heads over 128 values where items of few rows
// would spill: 64 sequences' own keys alone 45.5 us with one and 50.4 with two, fp32 queries 49.6 and
// 120, behind a prefix of 8,192 117 and 179; bf16 ones behind that prefix 99.4 and 84.6, which takes two.
template <int T, int DP, int RS, int RO>
constexpr int kWaves = DP <= 128 || RO == 64 || (RS == 64 && T != DQ_F32) ? 2 : 1;

// RS, RO: rows of the shared and of the own items' tiles.
template <int T, int TC, int DP, int DC, int RS, int RO>
__global__ __launch_bounds__(256, (kWaves<T, DP, RS, RO>)) void k_attn(AttnArgs a, AttnPart ws, AttnPart wo, int shared, int own) {
  __shared__ __align__(16) AttnLds<DP, RS> sh;
  // On every XCD a shared item for each of its 32 CUs, then an own one for each, and so on while both
  // last: a CU has a shared item, which computes, beside an own one, which reads.
  const int pairs = min(shared, own) / 256, b = blockIdx.x, turn = b / 256;
  const bool mixed = turn < 2 * pairs;
  const bool stacked = mixed ? turn % 2 == 0 : b - 256 * pairs < shared;
  const int of = mixed ? turn / 2 * 256 + b % 256 : stacked ? b - 256 * pairs : b - shared;
  const int index = xcd_item(of, stacked ? shared : own);
  if constexpr (RS == RO) {
    AttnPart w;
    w.tiles = stacked ? ws.tiles : wo.tiles;
    w.splits = stacked ? ws.splits : wo.splits;
    w.chunk = stacked ? ws.chunk : wo.chunk;
    w.slot = stacked ? ws.slot : wo.slot;
    w.own_from = wo.own_from;
    w.with_prefix = wo.with_prefix;
    w.backward = wo.backward;
    run_item<T, TC, DP, DC, RS>(a, w, stacked, index, sh);
  } else if (stacked) {
    run_item<T, TC, DP, DC, RS>(a, ws, true, index, sh);
  } else {
    run_item<T, TC, DP, DC, RO>(a, wo, false, index, sh);
  }
}

// ---- the join: the parts of a row, one wave a row ----------------------------

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

// Weights of up to 64 parts at a time lie one to a lane; their sums of v are read 8 at a time, the first 8 before
// anything is known of the row (a part that was not written is not used).
// Bound by two or three rounds of reads: 6.2 us for 2,048 rows of 9 parts of 128 values, 8.7 for 4,096 of 17 (36
// MB), 4 for a few rows; 16 parts at a time 1 us more.
template <int T, int TC>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, AttnPart wa, AttnPart wb) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  const int of = uniform((int)(id / a.heads)), h = uniform((int)(id % a.heads));
  const int t = first_token(a) + of;
  if (of >= a.part_tokens || t >= a.tokens) return;
  const int64_t R = (int64_t)a.part_tokens * a.group, step = R * a.cache.kv_heads;
  const int64_t at = (int64_t)(h / a.group) * R + (int64_t)of * a.group + h % a.group;
  const int d = 4 * lane, most = wa.splits + wb.splits;
  const bool in = d < a.dim;
  const float* po = a.part_o + at * a.dim + (in ? d : 0);
  v4f x[8];
  v2f ml = {-INFINITY, 0};
  auto read = [&](int s0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const v4f*>(po + min(s0 + i, most - 1) * step * a.dim);
  };
  auto read_ml = [&](int s0) {
    if (s0 + lane < most) ml = *reinterpret_cast<const v2f*>(a.part_ml + (at + (s0 + lane) * step) * 2);
  };
  read_ml(0);
  read(0);
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  // the own parts that were written: those that begin inside the sequence, and the first
  const int len = a.max_len > 0 ? min(max(a.lens[b], 0), a.max_len) : 0;
  const int end = wb.with_prefix ? (len > 0 ? wb.own_from + len : a.prefix_len) : len;
  const int own = wb.splits > 0 ? min(wb.splits, max(1, (end + wb.chunk - 1) / wb.chunk)) : 0;
  const int parts = wa.splits + own;
  float mx = -INFINITY, sum = 0;
  v4f y = {0, 0, 0, 0};
  for (int s0 = 0; s0 < parts; s0 += 64) {
    const int n = min(64, parts - s0);
    if (s0 > 0) read_ml(s0);
    const bool counts = lane < n;
    float top = counts ? ml[0] : -INFINITY;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
    top = fmaxf(top, mx);
    const float base = top == -INFINITY ? 0.f : top;
    const float f = counts ? exp2_fast(ml[0] - base) : 0.f, before = exp2_fast(mx - base);
    float l = counts ? ml[1] * f : 0.f;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) l += __shfl_xor(l, k, 64);
    sum = fmaf(sum, before, l);
    y *= before;
    mx = top;
    for (int s = 0; s < n; s += 8) {
      if (s0 + s > 0) read(s0 + s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float fi = as_f(__builtin_amdgcn_readlane(as_u(f), (s + i) & 63));
        if (s + i < n) y += x[i] * fi;  // (a factor of 0 too: what is infinite or NaN stays to be seen)
      }
    }
  }
  if (in) store4<T>(a, (int64_t)t * a.out_token + (int64_t)h * a.out_head, d, finish(y, sum, 1.f / sum));
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)t * a.heads + h] = lse_of(mx, sum, kShift<TC>);
}

template <int T, int TC, int DP, int DC, int RS, int RO>
hipError_t launch_items(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  const int64_t shared = (int64_t)p.shared.tiles * a.cache.kv_heads * p.shared.splits;
  const int64_t own = (int64_t)p.own.tiles * a.cache.kv_heads * p.own.splits * a.batch;
  hipLaunchKernelGGL((k_attn<T, TC, DP, DC, RS, RO>), dim3((uint32_t)(shared + own)), dim3(256), 0, s, a, p.shared, p.own,
                     (int)shared, (int)own);
  return hipGetLastError();
}

template <int T, int TC, int DP, int DC = DP>
hipError_t launch(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  const int rs = p.shared.splits > 0 ? p.shared.rows : p.own.rows, ro = p.own.rows;
  hipError_t e = hipErrorInvalidValue;
  if (rs == 16 && ro == 16) e = launch_items<T, TC, DP, DP, 16, 16>(a, p, s);
  if (rs == 64 && ro == 16) e = launch_items<T, TC, DP, DC, 64, 16>(a, p, s);
  if (rs == 64 && ro == 64) e = launch_items<T, TC, DP, DC, 64, 64>(a, p, s);
  if constexpr (T != DQ_F32 && DP <= 128) {
    if (rs == 128 && ro == 16) e = launch_items<T, TC, DP, DC, 128, 16>(a, p, s);
    if (rs == 128 && ro == 64) e = launch_items<T, TC, DP, DC, 128, 64>(a, p, s);
    if (rs == 128 && ro == 128) e = launch_items<T, TC, DP, DC, 128, 128>(a, p, s);
  }
  if (e != hipSuccess || a.part_o == nullptr) return e;
  hipLaunchKernelGGL((k_attn_join<T, TC>), dim3((uint32_t)(((int64_t)a.part_tokens * a.heads + 3) / 4)), dim3(256), 0, s, a, p.shared,
                     p.own);
  return hipGetLastError();
}

template <int T, int TC>
hipError_t by_dim(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  if (a.dim <= 64) return launch<T, TC, 64>(a, p, s);
  if (a.dim <= 96) return launch<T, TC, 128, 96>(a, p, s);
  if (a.dim <= 128) return launch<T, TC, 128>(a, p, s);
  if (a.dim <= 192) return launch<T, TC, 256, 192>(a, p, s);
  return launch<T, TC, 256>(a, p, s);
}

}  // namespace

hipError_t launch_attention(int type, int cache_type, const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  if (cache_type == DQ_F16) return type == DQ_F32 ? by_dim<DQ_F32, DQ_F16>(a, p, s) : by_dim<DQ_F16, DQ_F16>(a, p, s);
  return type == DQ_F32 ? by_dim<DQ_F32, DQ_BF16>(a, p, s) : by_dim<DQ_BF16, DQ_BF16>(a, p, s);
}

}  // namespace dq
