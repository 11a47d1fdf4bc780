// dq_pages.hip -- the pages that a query reads: each page's bounds of its keys' channels, the choice of pages
// by an upper bound of a row's scores on them, and attention over the chosen pages alone.
#include <algorithm>

#include "dq_attn_device.h"
#include "dq_pages.h"

namespace dq {
namespace {

// Row t of sequence b: the keys that it sees, the first of all.
DQ_DEV int row_sees(const AttnArgs& a, int b, int t, int len) {
  const int64_t end = a.q_offsets != nullptr ? a.q_offsets[b + 1] : t + 1;
  const int64_t n = len - end + t + 1;
  return (int)(n < 0 ? 0 : n < len ? n : len);
}

// Pages that hold a number of keys.
DQ_DEV int pages_of(int keys, int page_size) { return keys > 0 ? (keys - 1) / page_size + 1 : 0; }

// ---- bounds of a page -------------------------------------------------------
// A wave takes a page of a kv head: a lane 8 channels of every 64 / lanes'th key. 16-bit floats are compared as
// whole numbers of their order (negative ones with their other bits turned round), two at a time; NaN lies
// beyond the infinities there, at either end. Bound by the keys' bytes: 8 prompts of up to 16,384 keys, 8 f16 heads of 128 in pages
// of 16 (235 MB) 51 us, 4.6 TB/s; 64 pages of a decode step 5 us, a launch and three dependent reads.

typedef short v2s __attribute__((ext_vector_type(2)));

// The dword's two values as whole numbers that order as the values do, and back.
DQ_DEV u32 in_order(u32 x) { return x ^ (__builtin_bit_cast(u32, __builtin_bit_cast(v2s, x) >> 15) & 0x7FFF7FFFu); }
DQ_DEV u32 min2(u32 a, u32 b) {
  return __builtin_bit_cast(u32, __builtin_elementwise_min(__builtin_bit_cast(v2s, a), __builtin_bit_cast(v2s, b)));
}
DQ_DEV u32 max2(u32 a, u32 b) {
  return __builtin_bit_cast(u32, __builtin_elementwise_max(__builtin_bit_cast(v2s, a), __builtin_bit_cast(v2s, b)));
}

template <int TC>
__global__ __launch_bounds__(256) void k_page_bounds(AttnArgs a, const int32_t* from, int64_t slots, uint16_t* bounds, int lanes_log2,
                                                     int64_t item0, int64_t items) {
  const int lane = threadIdx.x & 63;
  const int64_t item = item0 + (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (item >= items) return;
  const CacheArgs& c = a.cache;
  const int h = (int)(item % c.kv_heads);
  const int64_t rest = item / c.kv_heads, slot = rest % slots;
  const int b = (int)(rest / slots);
  const int len = seq_len(a, b), start = from != nullptr ? min(max(from[b], 0), len) : 0;
  const int64_t p = start / c.page_size + slot;
  if (start >= len || p * c.page_size >= len) return;
  const int n = (int)min((int64_t)c.page_size, len - p * c.page_size);
  const int id = a.pages[b * a.pages_stride + p];
  if ((u32)id >= (u32)c.n_pages) return;
  const int lanes = 1 << lanes_log2, j = lane & (lanes - 1), step = 64 >> lanes_log2, d = 8 * j;
  const bool in = d < a.dim;
  const uint16_t* k = c.k + id * c.page + h * c.head + (in ? d : 0);
  v4u lo = {0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu}, hi = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
  constexpr int kLoads = 4;
  for (int i0 = 0; i0 < n; i0 += step * kLoads) {  // (lanes past the keys take the last again)
    v4u x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      x[u] = *reinterpret_cast<const v4u*>(k + (int64_t)min(i0 + u * step + (lane >> lanes_log2), n - 1) * c.token);
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32 y = in_order(x[u][e]);
        lo[e] = min2(lo[e], y);
        hi[e] = max2(hi[e], y);
      }
  }
  for (int m = lanes; m < 64; m <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = min2(lo[e], __shfl_xor(lo[e], m, 64));
      hi[e] = max2(hi[e], __shfl_xor(hi[e], m, 64));
    }
  constexpr int kInf = TC == DQ_F16 ? 0x7C00 : 0x7F80, kNan = TC == DQ_F16 ? 0x7E00 : 0x7FC0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    u32 l = in_order(lo[e]), u = in_order(hi[e]);
#pragma unroll
    for (int s = 0; s < 32; s += 16) {
      const int top = (int16_t)(hi[e] >> s), low = (int16_t)(lo[e] >> s);  // (-inf is ~kInf in that order)
      if (top > kInf || low < -kInf - 1) {
        l = (l & ~(0xFFFFu << s)) | ((u32)kNan << s);
        u = (u & ~(0xFFFFu << s)) | ((u32)kNan << s);
      }
    }
    lo[e] = l;
    hi[e] = u;
  }
  if (lane < lanes && in) {
    uint16_t* out = bounds + ((int64_t)id * c.kv_heads + h) * 2 * a.dim + d;
    *reinterpret_cast<v4u*>(out) = lo;
    *reinterpret_cast<v4u*>(out + a.dim) = hi;
  }
}

// ---- the choice of pages ----------------------------------------------------
// A row's score of a page is S = sum_d q+_d hi_d + q-_d lo_d, with q's positive values in q+ and the others in q-: a
// matrix product over 2 dim values, on the 16-bit matrix cores (an fp32 q in two parts). Two scores that differ must not tie for
// a rounding, so the choice is one of 64-bit sums; but of these it needs few. Beside S the same instructions give
// A = sum |q_d| max(|lo_d|, |hi_d|), with it a bound on S's error, and from both an interval that holds the 64-bit sum. A row's
// pages are certain where their intervals say so; only those that meet at the border of the choice (two or three of 512), and those whose sums
// are not finite, are summed again in 64 bits.
//
// 512 tokens of 32 heads on 512 pages of 4 kv heads of 128: scores 23 us, choice 14 (64-bit sums of all of them 479; as a library product in 64
// bits at 70 TFLOP/s, twice over the channels, 61). 32 sequences of up to 512 pages, 8 kv heads (51 MB of bounds), in one launch 18.6 us, 2.7
// TB/s: the reads take 11, then the choice of a row, some 7 us of dependent steps, which few waves hide.

constexpr uint64_t kAlways = ~0ull, kNanKey = ~0ull - 1;

DQ_DEV uint64_t order_key(double x) {
  if (x != x) return kNanKey;
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);  // (-0 is 0)
  return b >> 63 ? ~b : b | 1ull << 63;
}
DQ_DEV u32 order_key(float x) {
  const u32 b = as_u(x + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}

// The larger of a lane's and the one's 16 (32) lanes on.
DQ_DEV float pair_max16(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(as_u(x), as_u(x), false, false);
  return fmaxf(as_f(a[0]), as_f(a[1]));
}
DQ_DEV float pair_max32(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(as_u(x), as_u(x), false, false);
  return fmaxf(as_f(a[0]), as_f(a[1]));
}

template <int T>
constexpr int kScoreParts = T == DQ_F32 ? 2 : 1;

// What S may be off by, of A: a rounding (or a cut) of each of the 2 dim sums, A's own error, the interval's ends; with an fp32 q
// the sums of its second part, which are 2^-8 (f16: 2^-11) as large, and what two parts leave out of a value: 2^-18 (f16: 2^-22) of it.
template <int T, int TC>
DQ_DEV float score_error(int dim) {
  return (2 * dim + 64) * (T == DQ_F32 ? 0x1.04p-23f : 0x1p-23f) + (T != DQ_F32 ? 0.f : TC == DQ_F16 ? 0x1p-21f : 0x1p-17f);
}

// The bounds of 16 pages as B operands: lane n of a group has page n, 8 (lane / 16) .. + 7 of every 32 values.
template <int DP>
struct PageTile {
  v4u lo[DP / 32], hi[DP / 32];
  bool bad;
};
template <int DP>
DQ_DEV void load_page_tile(const AttnArgs& a, const ChooseArgs& c, int h, int id, int g, PageTile<DP>& p) {
  p.bad = (u32)id >= (u32)a.cache.n_pages;
  const uint16_t* near = c.bounds + ((int64_t)(p.bad ? 0 : id) * a.cache.kv_heads + h) * 2 * a.dim;
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) {
    const int d = 32 * s + 8 * g;
    p.lo[s] = d < a.dim ? *reinterpret_cast<const v4u*>(near + d) : v4u{0, 0, 0, 0};
    p.hi[s] = d < a.dim ? *reinterpret_cast<const v4u*>(near + a.dim + d) : v4u{0, 0, 0, 0};
  }
}
// The larger magnitudes of the bounds.
template <int DP>
DQ_DEV void magnitudes(const PageTile<DP>& p, v4u (&most)[DP / 32]) {
#pragma unroll
  for (int s = 0; s < DP / 32; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const v2us u = __builtin_bit_cast(v2us, p.lo[s][e] & 0x7FFF7FFFu), v = __builtin_bit_cast(v2us, p.hi[s][e] & 0x7FFF7FFFu);
      most[s][e] = __builtin_bit_cast(u32, __builtin_elementwise_max(u, v));
    }
}

// The intervals of the lane's page with rows 4 g .. + 3 of 16 query rows, where they pass low and high.
template <int T, int TC, int DP>
DQ_DEV void tile_scores(const RawQ<T, DP>& raw, const PageTile<DP>& page, const v4u (&most)[DP / 32], float error, int g, float (&low)[4],
                        float (&high)[4]) {
  constexpr int NS = DP / 32, NP = kScoreParts<T>;
  int e2 = 0;
  if constexpr (T == DQ_F32 && TC == DQ_F16) {  // scaled to a largest value in [2^14, 2^15)
    float top = 0;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(as_f(raw.x[s][i / 4][i % 4])));
    top = row_max(top);
    e2 = top > 0 && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
  }
  v4f sums[NP], size = {0, 0, 0, 0};
#pragma unroll
  for (int p = 0; p < NP; ++p) sums[p] = v4f{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    v4u part[NP], down, mag;  // down: the halves of values that are not above 0
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (T == DQ_F32) {
        const float y0 = ldexpf(as_f(raw.x[s][e / 2][e % 2 * 2]), e2), y1 = ldexpf(as_f(raw.x[s][e / 2][e % 2 * 2 + 1]), e2);
        u32 p = pack<TC>(y0, y1);
        part[0][e] = p;
        part[1][e] = pack<TC>(y0 - widen<TC>(p), y1 - widen_hi<TC>(p));
        down[e] = (y0 > 0 ? 0u : 0xFFFFu) | (y1 > 0 ? 0u : 0xFFFF0000u);
        // (what the parts leave out is less than 2^-17 (f16: 2^-21) of the value, or of the least magnitude that counts here)
        constexpr float kLeast = TC == DQ_F16 ? 0x1p-4f : 0x1p-100f;
        mag[e] = pack<TC>(y0 != y0 ? y0 : fmaxf(fabsf(y0), kLeast), y1 != y1 ? y1 : fmaxf(fabsf(y1), kLeast));
      } else {
        const u32 y = raw.x[s][0][e];
        part[0][e] = y;
        down[e] = __builtin_bit_cast(u32, __builtin_bit_cast(v2s, y) >> 15);
        mag[e] = y & 0x7FFF7FFFu;
      }
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      sums[p] = mma<TC>(part[p] & ~down, page.hi[s], sums[p]);
      sums[p] = mma<TC>(part[p] & down, page.lo[s], sums[p]);
    }
    size = mma<TC>(mag, most[s], size);
  }
  const v4f sum = NP == 1 ? sums[0] : sums[0] + sums[NP - 1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float d = fmaf(error, size[i], 0x1p-118f);
    const bool fine = d < INFINITY && fabsf(sum[i]) < INFINITY && !page.bad;
    const int back = T == DQ_F32 && TC == DQ_F16 ? -__shfl(e2, 4 * g + i, 64) : 0;
    low[i] = fmaxf(low[i], fine ? ldexpf(sum[i] - d, back) : -INFINITY);
    high[i] = fmaxf(high[i], fine ? ldexpf(sum[i] + d, back) : INFINITY);
  }
}

// The largest over a token's `rows` rows: of a lane's, then of two or all four lane groups.
DQ_DEV void token_max(float (&x)[4], int rows) {
  if (rows > 1) {
    x[0] = fmaxf(x[0], x[1]);
    x[2] = fmaxf(x[2], x[3]);
  }
  if (rows > 2) x[0] = fmaxf(x[0], x[2]);
  if (rows > 4) x[0] = pair_max16(x[0]);
  if (rows > 8) x[0] = pair_max32(x[0]);
}

// A wave takes 16 pages of a kv head, whose bounds it holds, and of a sequence's rows a range, 16 at a time: `slots` tokens
// of 2^rows_log2 rows, a power of two of at least the kv head's query heads (16 where they are more: one 16 after the other).
// The four waves of a workgroup take 64 pages in a row and read the same rows: each loads a part of the next ones, all take them from LDS
// (a row's 16 bytes a lane are lines of 16 rows at once, slow to ask for; every wave for itself 41.4 us against 37.9 of scores and choice below,
// with fp32 rows 72 against 59).
template <int T, int TC, int DP>
__global__ __launch_bounds__(256, 2) void k_page_scores(AttnArgs a, ChooseArgs c, int token0, int rows_log2, int ranges, int range_tokens) {
  constexpr int K = T == DQ_F32 ? 2 : 1, kLoads = DP / 32 * K;  // 16 bytes a lane, of 16 rows
  constexpr int kMine = (kLoads + 3) / 4;                       // of a wave
  __shared__ v4u sh[2][kLoads][64];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wave = uniform(threadIdx.x >> 6);
  const int hk = a.cache.kv_heads, page_groups = (c.pages + 63) / 64;
  u32 item = blockIdx.x;
  const int group0 = (int)(item % page_groups) * 64, p0 = group0 + 16 * wave;
  item /= page_groups;
  const int h = item % hk;
  item /= hk;
  const int range = item % ranges, b = item / ranges;
  // the range's tokens, of the launch's (offsets, length and page numbers under way together)
  const int64_t lo = a.q_offsets != nullptr ? a.q_offsets[b] : b, hi = a.q_offsets != nullptr ? a.q_offsets[b + 1] : b + 1;
  // (the last sequence's list may end with its keys)
  const int32_t* list = a.pages + b * a.pages_stride;
  int listed = 0;
  if (b + 1 < a.batch) listed = list[min(p0 + n, c.pages - 1)];
  const int pages = pages_of(seq_len(a, b), a.cache.page_size);
  if (b + 1 == a.batch && p0 + n < pages) listed = list[p0 + n];
  const int64_t end = min(min(hi, (int64_t)a.tokens), (int64_t)token0 + c.tokens);
  const int64_t first = max(lo, (int64_t)token0) + (int64_t)range * range_tokens, last = min(first + range_tokens, end);
  if (group0 >= pages || first >= last) return;
  const int rows = 1 << rows_log2, slots = 16 >> rows_log2, slot = n >> rows_log2, blocks = (a.group + 15) / 16;
  v4u mine[kMine];
  auto read = [&](int64_t t0, int block) {  // (a row past the heads is the last again)
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int load = 4 * j + wave;
      if (kLoads % 4 == 0 || load < kLoads)
        mine[j] = load_q16<T>(a, (int)min(t0 + slot, last - 1), h * a.group + min(16 * block + (n & (rows - 1)), a.group - 1),
                              32 * (load / K) + 8 * g, load % K);
    }
  };
  auto share = [&](int at) {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int load = 4 * j + wave;
      if (kLoads % 4 == 0 || load < kLoads) sh[at][load][lane] = mine[j];
    }
    __syncthreads();
  };
  read(first, 0);
  PageTile<DP> page;
  load_page_tile<DP>(a, c, h, p0 + n < pages ? listed : 0, g, page);
  share(0);
  v4u most[DP / 32];
  magnitudes<DP>(page, most);
  const float error = score_error<T, TC>(a.dim);
  int at = 0;
  for (int64_t t0 = first; t0 < last; t0 += slots) {
    float low[4], high[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) low[i] = high[i] = -INFINITY;
    for (int block = 0; block < blocks; ++block) {
      const bool same = block + 1 < blocks;
      const int64_t t1 = same ? t0 : t0 + slots;
      if (t1 < last) read(t1, same ? block + 1 : 0);
      if (p0 < pages) {
        RawQ<T, DP> raw;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) raw.x[i / K][i % K] = sh[at][i][lane];
        tile_scores<T, TC, DP>(raw, page, most, error, g, low, high);
      }
      at ^= 1;
      if (t1 < last) share(at);  // (read a tile ago, before the last barrier)
    }
    if (p0 >= pages) continue;
    token_max(low, rows);
    token_max(high, rows);
    uint64_t* out = c.keys + ((t0 - token0) * hk + h) * c.pages + p0 + n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * g + i, to = row >> rows_log2;
      if ((row & (rows - 1)) == 0 && t0 + to < last && p0 + n < pages) *reinterpret_cast<v2f*>(out + (int64_t)to * hk * c.pages) = v2f{low[i], high[i]};
    }
  }
}

template <int kCtrl>
DQ_DEV double dpp_add(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint64_t o = (uint64_t)(u32)dpp<kCtrl>((int)(b >> 32)) << 32 | (u32)dpp<kCtrl>((int)b);
  return x + __builtin_bit_cast(double, o);
}
// The sum over each aligned group of 2^log2 lanes.
DQ_DEV double lanes_sum(double x, int log2) {
  if (log2 >= 1) x = dpp_add<kQuadXor1>(x);
  if (log2 >= 2) x = dpp_add<kQuadXor2>(x);
  if (log2 >= 3) x = dpp_add<kHalfMirror>(x);
  if (log2 >= 4) x = dpp_add<kRowRor8>(x);
  if (log2 >= 5) x += __shfl_xor(x, 16, 64);
  return x;
}

// The 64-bit scores of row t's query heads on `count` pages id_of(j), as whole numbers that order as they do: most[j] (in LDS, 0 before)
// is the largest over the heads. A wave's work: every `step`th, from its `first` on, of the steps of a page and 64 / 2^log2
// of its heads; N steps' loads are under way together (one step's after the other's, a row with an open page waits 1 us longer).
template <int T, int TC, int N = 4, class F>
DQ_DEV void exact_keys(const AttnArgs& a, const ChooseArgs& c, int t, int h, int count, F&& id_of, uint64_t* most, int first, int step, int log2,
                       int lane) {
  const int lanes = 1 << log2, d = 8 * (lane & (lanes - 1)), at_once = 64 >> log2, turns = (a.group + at_once - 1) / at_once;
  const bool in = d < a.dim;
  const int steps = count * turns;
  for (int i0 = first * N; i0 < steps; i0 += step * N) {
    v4u lo[N], hi[N], x[N][T == DQ_F32 ? 2 : 1];
    int page[N];
    bool bad[N];
    int64_t at[N];
    int p = i0 / turns, turn = i0 - p * turns;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      page[k] = p;
      const int head = min(turn * at_once + (lane >> log2), a.group - 1);
      at[k] = (int64_t)t * a.q_token + (int64_t)(h * a.group + head) * a.q_head + (in ? d : 0);
      const int id = id_of(p);
      bad[k] = (u32)id >= (u32)a.cache.n_pages;
      const uint16_t* near = c.bounds + ((int64_t)(bad[k] ? 0 : id) * a.cache.kv_heads + h) * 2 * a.dim + (in ? d : 0);
      lo[k] = *reinterpret_cast<const v4u*>(near);
      hi[k] = *reinterpret_cast<const v4u*>(near + a.dim);
      if (i0 + k + 1 < steps && ++turn == turns) {  // (past the steps: the last again)
        turn = 0;
        ++p;
      }
    }
    load8s<T>(a, at, x);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (k > 0 && i0 + k >= steps) break;
      double s[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = T == DQ_F32 ? as_f(x[k][e / 4 % (T == DQ_F32 ? 2 : 1)][e % 4]) : e % 2 ? widen_hi<T>(x[k][0][e / 2]) : widen<T>(x[k][0][e / 2]);
        const u32 y = q > 0 ? hi[k][e / 2] : lo[k][e / 2];
        s[e % 2] = fma((double)q, (double)(e % 2 ? widen_hi<TC>(y) : widen<TC>(y)), s[e % 2]);
      }
      const uint64_t key = order_key(lanes_sum(in ? s[0] + s[1] : 0.0, log2));
      if ((lane & (lanes - 1)) == 0) atomicMax((unsigned long long*)&most[page[k]], (unsigned long long)(bad[k] ? kNanKey : key));
    }
  }
}

// Keys of all of a row's pages in 64 bits, where too many meet at the border: they take the intervals' place.
DQ_DEV uint64_t load_key(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DQ_DEV void store_key(uint64_t* p, uint64_t x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The choice: W waves take a row's kv head. The count-th largest of the intervals' ends is found bit by bit, on whole numbers that
// order as they do. kHeld: a row's intervals lie in registers, N to a lane (`held`), else they are read again for every bit. Wave w takes
// a run of the pages, so that the list comes out ascending. exact(n) sums the scores of the n open pages in sh.list into sh.key;
// it is called once for a row with more pages than it reads.
template <int W>
struct ChoiceLds {
  int counts[2][W], list[64];
  uint64_t key[64];
};

template <int T, int TC, int N, int W, bool kHeld, class F>
DQ_DEV void choose_row(const AttnArgs& a, const ChooseArgs& c, int t, int h, int b, int pages, uint64_t* keys, const v2f (&held)[N], ChoiceLds<W>& sh,
                       int w, int lane, int log2, F&& exact) {
  auto &s_counts = sh.counts;
  auto &s_list = sh.list;
  auto &s_key = sh.key;
  const int hk = a.cache.kv_heads;
  int32_t* out = c.chosen + ((int64_t)t * hk + h) * c.count;
  const int count = (int)min(c.count, (int64_t)pages), tid = w * 64 + lane;
  for (int64_t i = count + tid; i < c.count; i += 64 * W) out[i] = -1;
  if (pages <= c.count) {
    for (int i = tid; i < pages; i += 64 * W) out[i] = i;
    return;
  }
  const int32_t* list = a.pages + b * a.pages_stride;
  int number[N];  // of the pages held
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < N; ++i) number[i] = list[min((w * N + i) * 64 + lane, pages - 1)];
  }
  const int rounds = kHeld ? N : (pages + 64 * W - 1) / (64 * W), base = w * rounds * 64;
  auto interval = [&](int i, v2f x, u32& low, u32& high) {
    const int p = base + i * 64 + lane;
    const bool always = p < c.first || p >= pages - c.last;
    low = p >= pages ? 0u : always ? ~0u : order_key(x[0]);  // (0: no page)
    high = p >= pages ? 0u : always ? ~0u : order_key(x[1]);
  };
  u32 low[N], high[N];
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < N; ++i) interval(i, held[i], low[i], high[i]);
  }
  // the sum over the row's waves
  int turn = 0;
  auto all_waves = [&](int n) {
    if constexpr (W == 1) return n;
    turn ^= 1;
    if (lane == 0) s_counts[turn][w] = n;
    __syncthreads();  // (a turn's counts are read before the next one's barrier, written after it)
    int sum = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) sum += s_counts[turn][i];
    return sum;
  };
  // f(round, low, high) for the wave's pages
  auto each = [&](auto&& f) {
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < N; ++i) f(i, low[i], high[i]);
    } else {
      for (int i = 0; i < rounds; ++i) {
        u32 l, u;
        interval(i, *reinterpret_cast<const v2f*>(keys + min(base + i * 64 + lane, c.pages - 1)), l, u);
        f(i, l, u);
      }
    }
  };
  // the least over the row's waves
  auto all_least = [&](u32 x) {
    x = wave_least(x);
    if constexpr (W == 1) return x;
    turn ^= 1;
    if (lane == 0) s_counts[turn][w] = (int)x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) x = min(x, (u32)s_counts[turn][i]);
    return x;
  };
  // the n-th largest low (high) end, of values from `bottom` to `top` (and pages of ~0, which are above); early: or a lower
  // value with n ends above it or at it
  auto nth = [&](int n, u32 bottom, u32 top, bool highs, bool early) {
    int bit = 31 - __builtin_clz((bottom ^ top) | 1);
    u32 least = top & ~((2u << bit) - 1);
    int taken = 0;
#pragma unroll 1
    for (; bit >= 0 && !(early && taken == n); --bit) {
      const u32 mid = least | 1u << bit;
      int k = 0;
      each([&](int, u32 l, u32 u) { k += __popcll(__ballot((highs ? u : l) >= mid)); });
      k = all_waves(k);
      if (k >= n) {
        least = mid;
        taken = k;
      }
    }
    return least;
  };
  // A page whose high end is below the count-th largest low end is out; one whose low end is above the next high
  // end after the count-th is in; the others are open.
  u32 bottom = ~0u, top = 0;
  each([&](int, u32 l, u32) {
    if (l != 0) bottom = min(bottom, l);
    if (l != ~0u) top = max(top, l);
  });
  bottom = all_least(bottom);
  top = ~all_least(~top);
  const u32 floor = count <= c.first + c.last ? ~0u : nth(count, bottom, top, false, true);
  int able = 0;
  each([&](int, u32, u32 u) { able += __popcll(__ballot(u >= floor)); });
  able = all_waves(able);
  u32 ceiling = 0;
  int over = able - count;  // the next high end is the over-th least of those able
  if (over > 0 && over <= 8) {
    u32 from = floor;
    while (true) {
      u32 least = ~0u;
      each([&](int, u32, u32 u) {
        if (u >= from) least = min(least, u);
      });
      least = all_least(least);
      int same = 0;
      each([&](int, u32, u32 u) { same += __popcll(__ballot(u == least)); });
      over -= all_waves(same);
      ceiling = least;
      if (over <= 0) break;
      from = least + 1;
    }
  } else if (over > 0) {
    ceiling = nth(count + 1, 0u, ~1u, true, false);
  }
  const bool all_in = able == count;
  int open = 0;
  if (!all_in) each([&](int, u32 l, u32 u) { open += __popcll(__ballot(u >= floor && l <= ceiling)); });
  open = all_waves(open);
  int before = 0;  // open ones of the waves before
  if constexpr (W > 1)
    for (int i = 0; i < w; ++i) before += s_counts[turn][i];
  const int room = count - (able - open);  // for open ones
  uint64_t taken = 0;  // of the open ones, in their order
  const int looked = open <= 64 ? open : 0;
  if (looked > 0) {
    int at = before;
    s_key[lane] = 0;  // (of all waves alike)
    each([&](int i, u32 l, u32 u) {
      const bool mine = u >= floor && l <= ceiling;
      const uint64_t m = __ballot(mine);
      if (mine) s_list[at + __popcll(m & ((1ull << lane) - 1))] = kHeld ? number[kHeld ? i : 0] : list[base + i * 64 + lane];
      at += __popcll(m);
    });
    if constexpr (W > 1) __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  }
  exact(looked);
  if (looked > 0) {
    if constexpr (W > 1) __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    const uint64_t key = lane < open ? s_key[lane] : 0;
    int rank = 0;
    for (int j = 0; j < open; ++j) {
      const uint64_t o = s_key[j];
      rank += o > key || (o == key && j < lane);
    }
    taken = __ballot(lane < open && rank < room);
  } else if (open > 64) {
    for (int p0 = 0; p0 < pages; p0 += 64) {
      const int some = min(64, pages - p0);
      s_key[lane] = 0;
      if constexpr (W > 1) __syncthreads();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
      exact_keys<T, TC>(a, c, t, h, some, [&](int j) { return list[p0 + j]; }, s_key, w, W, log2, lane);
      if constexpr (W > 1) __syncthreads();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
      const int p = p0 + lane;
      if (w == 0 && lane < some) store_key(keys + p, p < c.first || p >= pages - c.last ? kAlways : s_key[lane]);
      if constexpr (W > 1) __syncthreads();
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "agent");
    if constexpr (W > 1) __syncthreads();
    auto key_at = [&](int i) {
      const int p = base + i * 64 + lane;
      return p < pages ? load_key(keys + p) : 0;
    };
    uint64_t least = 0;
    int k = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0 && k != count; --bit) {
      const uint64_t mid = least | 1ull << bit;
      int m = 0;
      for (int i = 0; i < rounds; ++i) m += __popcll(__ballot(key_at(i) >= mid));
      m = all_waves(m);
      if (m >= count) {
        least = mid;
        k = m;
      }
    }
    int above = 0, ties = 0;
    for (int i = 0; i < rounds; ++i) {
      above += __popcll(__ballot(key_at(i) > least));
      ties += __popcll(__ballot(key_at(i) == least));
    }
    const int all_above = all_waves(above);
    int at = 0, left = count - all_above, ties_before = 0;
    if constexpr (W > 1) {
      for (int i = 0; i < w; ++i) at += s_counts[turn][i];
      all_waves(ties);
      for (int i = 0; i < w; ++i) ties_before += s_counts[turn][i];
    }
    at += min(ties_before, left);
    left = max(left - ties_before, 0);
    for (int i = 0; i < rounds; ++i) {
      const uint64_t key = key_at(i), tie = __ballot(key == least), lower = (1ull << lane) - 1;
      const bool mine = key > least || (key == least && __popcll(tie & lower) < left);
      const uint64_t m = __ballot(mine);
      if (mine) out[at + __popcll(m & lower)] = base + i * 64 + lane;
      at += __popcll(m);
      left -= min(left, __popcll(tie));
    }
    return;
  }
  // certain ones and taken ones, in their order
  int sure = 0;
  each([&](int, u32 l, u32 u) { sure += __popcll(__ballot(u >= floor && (all_in || l > ceiling))); });
  int at = before < 64 ? __popcll(taken & ((1ull << before) - 1)) : __popcll(taken), seen = before;
  if constexpr (W > 1) {
    all_waves(sure);
    for (int i = 0; i < w; ++i) at += s_counts[turn][i];
  }
  each([&](int i, u32 l, u32 u) {
    const uint64_t lower = (1ull << lane) - 1;
    const bool isopen = !all_in && u >= floor && l <= ceiling;
    const uint64_t mo = __ballot(isopen);
    const int index = seen + __popcll(mo & lower);
    const bool mine = isopen ? taken >> index & 1 : u >= floor;
    const uint64_t m = __ballot(mine);
    if (mine) out[at + __popcll(m & lower)] = base + i * 64 + lane;
    at += __popcll(m);
    seen += __popcll(mo);
  });
}

// W 1: four rows a workgroup.
template <int T, int TC, int N, int W, bool kHeld>
__global__ __launch_bounds__(W == 1 ? 256 : W * 64) void k_page_choice(AttnArgs a, ChooseArgs c, int token0, int64_t rows, int log2) {
  constexpr int R = W == 1 ? 4 : 1;  // rows of a workgroup
  __shared__ ChoiceLds<W> sh[R];
  const int lane = threadIdx.x & 63, hk = a.cache.kv_heads;
  const int in_group = uniform(threadIdx.x >> 6), w = W == 1 ? 0 : in_group, r = W == 1 ? in_group : 0;
  const int64_t row = (int64_t)blockIdx.x * R + r;
  if (row >= rows) return;
  const int t = token0 + (int)(row / hk), h = (int)(row % hk);
  uint64_t* keys = c.keys + row * c.pages;
  v2f held[N];  // the intervals, under way before anything is known of the row
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      held[i] = c.keys != nullptr ? *reinterpret_cast<const v2f*>(keys + min((w * N + i) * 64 + lane, c.pages - 1)) : v2f{0, 0};
  }
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  const int pages = pages_of(row_sees(a, b, t, seq_len(a, b)), a.cache.page_size);
  choose_row<T, TC, N, W, kHeld>(a, c, t, h, b, pages, keys, held, sh[r], w, lane, log2, [&](int n) {
    exact_keys<T, TC>(a, c, t, h, n, [&](int j) { return sh[r].list[j]; }, sh[r].key, w, W, log2, lane);
  });
}

// Both steps in one launch, for few rows: a workgroup's waves score a row's pages, 16 each in turn, into LDS; the first wave
// chooses, all sum what is open.
constexpr int kPickPages = 512;

template <int T, int TC, int DP>
__global__ __launch_bounds__(DP <= 128 ? 1024 : 512) void k_page_pick(AttnArgs a, ChooseArgs c, int token0, int log2) {
  constexpr int kWaves = DP <= 128 ? 16 : 8, N = kPickPages / 64;
  __shared__ ChoiceLds<1> sh;
  __shared__ v2f s_scores[kPickPages];
  __shared__ int s_open;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), hk = a.cache.kv_heads;
  const int n = lane & 15, g = lane >> 4;
  const int h = (int)(blockIdx.x % hk), t = token0 + (int)(blockIdx.x / hk);
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  const int blocks = (a.group + 15) / 16;
  RawQ<T, DP> raw;
  load_q<T, DP>(a, true, t, h * a.group + min(n, a.group - 1), g, raw);  // (a row past the heads is the last again)
  const int32_t* list = a.pages + b * a.pages_stride;
  const int pages = pages_of(row_sees(a, b, t, seq_len(a, b)), a.cache.page_size);
  if (pages > c.count) {
    const float error = score_error<T, TC>(a.dim);
    for (int p0 = 16 * wave; p0 < pages; p0 += 16 * kWaves) {
      PageTile<DP> page;
      load_page_tile<DP>(a, c, h, p0 + n < pages ? list[p0 + n] : 0, g, page);
      v4u most[DP / 32];
      magnitudes<DP>(page, most);
      float low[4], high[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) low[i] = high[i] = -INFINITY;
      for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load_q<T, DP>(a, true, t, h * a.group + min(16 * block + n, a.group - 1), g, raw);
        tile_scores<T, TC, DP>(raw, page, most, error, g, low, high);
      }
      token_max(low, 16);
      token_max(high, 16);
      if (g == 0 && p0 + n < pages) s_scores[p0 + n] = v2f{low[0], high[0]};
    }
  }
  __syncthreads();
  // all waves sum what is open
  auto exact = [&](int n) {
    if (wave == 0 && lane == 0) s_open = n;
    __syncthreads();
    exact_keys<T, TC, 1>(a, c, t, h, s_open, [&](int j) { return sh.list[j]; }, sh.key, wave, kWaves, log2, lane);
    __syncthreads();
  };
  if (wave > 0) {
    if (pages > c.count) exact(0);
    return;
  }
  v2f held[N];
#pragma unroll
  for (int i = 0; i < N; ++i) held[i] = s_scores[i * 64 + lane];
  choose_row<T, TC, N, 1, true>(a, c, t, h, b, pages, c.keys + ((int64_t)(t - token0) * hk + h) * c.pages, held, sh, 0, lane, log2, exact);
}

// ---- attention over chosen pages ---------------------------------------------
// An item is (token, kv head, up to 16 of its query heads, range of the list): its rows see the same keys. The four
// waves take 32 keys each in turn, with a running softmax of their own, and add up at the end. Scores are S^T = K
// Q^T, which leaves a lane with the weights that O^T = V^T P^T takes from it. Loads take 16 bytes a lane and whole lines a
// row of lanes: of values a lane holds DP / 16 of 8 keys, as O^T takes them; of keys S^T takes 8 values of one key a
// lane, 16 keys a row of lanes, so they turn in LDS, a wave's own part of it (16 bytes of a key at a place turned by the key's number: no two of
// a read meet in a bank). The next tile's keys are under way from when this one's are in LDS.
//
// 32 sequences of 4,096 chosen keys, 32 / 8 bf16 heads of 128 (537 MB): 92 to 112 us with the pages' place in memory, 4.8 to 5.8 TB/s (a part of
// them from the cache behind the L2s).
// 473 rows of 1,024 chosen keys each, two sequences of up to 8,192: 86 us; 2 GB come from the L2s (93% hits), 23 TB/s. With one-part weights 81: then keys
// loaded in S^T's order, whose neighbouring lanes read 16 lines, took 137 us; turned, not asked for early 86; rows of sums not turned in LDS 84.

template <int DP>
struct PageLds {
  union alignas(16) {  // of a wave
    v4u k[32][DP / 8];
    v4f o[16][DP / 4];  // (a row's turned by its number)
  } own[4];
  float ml[4][16][2];
  int bad;
};

template <int DP>
struct PageKv {
  v4u k[2][DP / 32];
  u32 v[8][DP / 32];
};

// Where the lane goes if those of `first`, then those of `second`, then the others are lined up.
DQ_DEV int front_place(uint64_t first, uint64_t second, int lane) {
  const uint64_t lower = (1ull << lane) - 1;
  if (first >> lane & 1) return __popcll(first & lower);
  if (second >> lane & 1) return __popcll(first) + __popcll(second & lower);
  return __popcll(first | second) + __popcll(~(first | second) & lower);
}

// Two weights of a 16-bit row, each in two parts: the first is cut, so that neither is negative and an infinite value of a
// key that has a weight stays what it is. Together they are within 2^-16 (f16: 2^-22, and 2^-24 in all) of the weight; one rounded part
// (2^-8, 2^-11) puts outputs off by up to a rounding of theirs. Both / one, us, 32 / 8 bf16 heads of 64, 128, 256: 32 sequences of 4,096 chosen
// keys 42 / 42, 107 / 106, 202 / 202; 473 rows of 1,024 chosen keys 59 / 54, 86 / 82, 241 / 226.
template <int TC>
DQ_DEV void split_weights(float a, float b, u32 (&out)[2]) {
  if constexpr (TC == DQ_F16) {
    out[0] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(a, b));
    out[1] = pack<TC>(fmaxf(a - widen<TC>(out[0]), fminf(a, 0x1p-24f)), fmaxf(b - widen_hi<TC>(out[0]), fminf(b, 0x1p-24f)));
  } else {
    out[0] = __builtin_amdgcn_perm(as_u(b), as_u(a), 0x07060302u);
    out[1] = pack<TC>(fmaxf(a - widen<TC>(out[0]), 0x1p-17f * a), fmaxf(b - widen_hi<TC>(out[0]), 0x1p-17f * b));
  }
}

template <int T, int TC, int DP>
__global__ __launch_bounds__(256, (T != DQ_F32 && DP <= 128 ? 3 : 1)) void k_page_attn(AttnArgs a, const int32_t* chosen, int64_t count, int splits, int chunk, int tiles) {
  constexpr int NP = kParts<T, TC>, NW = T == DQ_F32 ? NP : 2;  // parts of a query, of a weight
  constexpr int NC = DP / 16;
  __shared__ PageLds<DP> sh;
  const CacheArgs& ca = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  u32 item = blockIdx.x;
  const int head = item % ca.kv_heads;
  item /= ca.kv_heads;
  const int tile0 = item % tiles * 16;
  item /= tiles;
  const int range = item % splits, t = item / splits;
  const int rows = min(16, a.group - tile0);
  const int64_t e0 = (int64_t)range * chunk, e1 = min(e0 + chunk, count);
  const int32_t* list = chosen + ((int64_t)t * ca.kv_heads + head) * count;
  // (the list, the queries and the sequence under way together)
  int entry = e0 + lane < e1 ? list[e0 + lane] : -1;
  RawQ<T, DP> raw;
  load_q<T, DP>(a, n < rows, t, head * a.group + tile0 + min(n, rows - 1), g, raw);
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  if (threadIdx.x == 0) sh.bad = 0;
  __syncthreads();
  const int sees = row_sees(a, b, t, seq_len(a, b));
  v4u q[NP][DP / 32];
  const float c = q_operands<T, TC, DP>(a, raw, q);

  RowMax rm;
  float l = 0;
  v4f o[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i] = v4f{0, 0, 0, 0};
  bool bad = false;

  const u32 token_bytes = (u32)ca.token * 2;
  constexpr u32 kOut = 0x80000000u;  // an offset past every buffer: such loads give 0
  constexpr int kChunks = DP / 8, kLine = 64 / kChunks;  // 16 bytes, of a key; keys of a load
  constexpr int kTurn = kChunks < 16 ? 7 : 15;
  const int key0 = lane / kChunks, chunk0 = lane % kChunks;
  const u32 koff = 8 * chunk0 < a.dim ? key0 * token_bytes + 16 * chunk0 : kOut;
  auto& ktile = sh.own[wave].k;
  u32 voff[DP / 128 > 0 ? DP / 128 : 1];
#pragma unroll
  for (int s = 0; s < (DP / 128 > 0 ? DP / 128 : 1); ++s) {
    const int d = n * NC + 8 * s;
    voff[s] = d < a.dim ? 4 * g * token_bytes + d * 2 : kOut;
  }

  const int units = ca.page_size / 16;  // of 16 keys, of a page
  const int skip = 8 / units, skip_rest = 8 % units;
  for (int64_t eb = e0; eb < e1; eb += 64) {
    // the next 64 entries, a lane each; those that hold visible keys to the front
    if (eb > e0) entry = eb + lane < e1 ? list[eb + lane] : -1;
    const bool some = entry >= 0 && (int64_t)entry * ca.page_size < sees;
    int id = some ? a.pages[b * a.pages_stride + entry] : 0;
    if (some && (u32)id >= (u32)ca.n_pages) {
      bad = true;
      id = 0;
    }
    // (the page of the last visible key, which may hold few, at the end of them)
    const int seen = some ? min((sees - entry * ca.page_size + 15) / 16, units) : 0;  // 16s of keys
    const uint64_t full = __ballot(seen == units), part = __ballot(some && seen < units);
    const int left = units - (part != 0 ? __builtin_amdgcn_readlane(seen, 63 - __builtin_clzll(part)) : units);
    const int to = front_place(full, part, lane);
    entry = __builtin_amdgcn_ds_permute(4 * to, entry);
    id = __builtin_amdgcn_ds_permute(4 * to, id);
    const int halves = __popcll(full | part) * units - left;  // of tiles: runs of 16 keys
    int e = 2 * wave / units, sub = 2 * wave % units;
    // the tile at `half`: its keys' first indexes and places; its keys are asked for (past the end nothing is)
    PageKv<DP> r;
    int kb[2], kb_next[2];
    int64_t base[2], base_next[2];
    auto next = [&](int half) {
      const int id0 = __builtin_amdgcn_readlane(id, e);
      kb_next[0] = __builtin_amdgcn_readlane(entry, e) * ca.page_size + 16 * sub;
      base_next[0] = id0 * ca.page + 16 * sub * ca.token + head * ca.head;
      kb_next[1] = INT32_MAX - 16;  // (no key)
      base_next[1] = base_next[0];
      if (half + 1 < halves) {
        const bool over = sub + 1 == units;
        const int e2 = over ? e + 1 : e, sub2 = over ? 0 : sub + 1;
        kb_next[1] = __builtin_amdgcn_readlane(entry, e2) * ca.page_size + 16 * sub2;
        base_next[1] = __builtin_amdgcn_readlane(id, e2) * ca.page + 16 * sub2 * ca.token + head * ca.head;
      }
      e += skip;
      sub += skip_rest;
      if (sub >= units) {
        sub -= units;
        ++e;
      }
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const auto kr = rsrc(ca.k + base_next[t2], half < halves ? 0x7FFFFFFFu : 0u);
#pragma unroll
        for (int s = 0; s < DP / 32; ++s)
          r.k[t2][s] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(kr, koff, s * kLine * token_bytes, 0));
      }
    };
    next(2 * wave);
    for (int half = 2 * wave; half < halves; half += 8) {
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        kb[t2] = kb_next[t2];
        base[t2] = base_next[t2];
      }
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const auto vr = rsrc(ca.v + base[t2], 0x7FFFFFFFu);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (DP == 64) {
            const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_raw_buffer_load_b64(vr, voff[0], i * token_bytes, 0));
            r.v[4 * t2 + i][0] = x[0];
            r.v[4 * t2 + i][1] = x[1];
          } else {
#pragma unroll
            for (int s = 0; s < DP / 128; ++s) {
              const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[s], i * token_bytes, 0));
#pragma unroll
              for (int w = 0; w < 4; ++w) r.v[4 * t2 + i][4 * s + w] = x[w];
            }
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) {
          const int key = key0 + s * kLine;
          ktile[16 * t2 + key][chunk0 ^ (key & kTurn)] = r.k[t2][s];
        }
      __builtin_amdgcn_wave_barrier();
      next(half + 8);
      float x[8];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        v4u k[DP / 32];
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) k[s] = ktile[16 * t2 + n][(4 * s + g) ^ (n & kTurn)];
        v4f acc = {0, 0, 0, 0};
#pragma unroll
        for (int p = NP - 1; p >= 0; --p)
#pragma unroll
          for (int s = 0; s < DP / 32; ++s) acc = mma<TC>(k[s], q[p][s], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * t2 + i] = acc[i];
      }
      if (kb[0] + 16 > sees || kb[1] + 16 > sees) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool hidden = kb[j >> 2] + 4 * g + (j & 3) >= sees;
          x[j] = hidden ? -INFINITY : x[j];
#pragma unroll
          for (int w = 0; w < DP / 32; ++w)
            if (hidden) r.v[j][w] = 0;  // places past the keys may hold anything
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
      v4u p[NW];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32 parts[NW];
        if constexpr (T == DQ_F32)
          split<T, TC>(x[2 * j], x[2 * j + 1], parts);
        else
          split_weights<TC>(x[2 * j], x[2 * j + 1], parts);
#pragma unroll
        for (int k = 0; k < NW; ++k) p[k][j] = parts[k];
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        v4u vt;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          vt[w] = __builtin_amdgcn_perm(r.v[2 * w + 1][i >> 1], r.v[2 * w][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int k = NW - 1; k >= 0; --k) o[i] = mma<TC>(vt, p[k], o[i]);
      }
    }
  }

  // the waves' sums join in LDS
  l = row_sum(l);
  if (g == 0) {
    sh.ml[wave][n][0] = rm.m;
    sh.ml[wave][n][1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = (4 * g + i) * NC;
#pragma unroll
    for (int w = 0; w < NC / 4; ++w) sh.own[wave].o[n][(d / 4 + w) ^ n] = v4f{o[4 * w][i], o[4 * w + 1][i], o[4 * w + 2][i], o[4 * w + 3][i]};
  }
  if (bad) sh.bad = 1;
  __syncthreads();
  const int quads = a.dim / 4;
  for (int i = threadIdx.x; i < rows * quads; i += 256) {
    const int r = i / quads, d4 = i % quads;
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) mx = fmaxf(mx, sh.ml[k][r][0]);
    v4f y = {0, 0, 0, 0};
    float sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float mk = sh.ml[k][r][0];
      const float f = mk == -INFINITY ? 0.f : exp2_fast(mk - mx);
      sum = fmaf(sh.ml[k][r][1], f, sum);
      y += sh.own[k].o[r][d4 ^ r] * f;
    }
    if (sh.bad) sum = __builtin_nanf("");
    const int h = head * a.group + tile0 + r;
    if (a.part_o == nullptr) {
      store4<T>(a, (int64_t)t * a.out_token + (int64_t)h * a.out_head, 4 * d4, finish(y, sum, 1.f / sum));
      if (a.lse != nullptr && d4 == 0) a.lse[(int64_t)t * a.heads + h] = lse_of(mx, sum, kShift<TC>);
    } else {
      const int64_t at = ((int64_t)range * ca.kv_heads + head) * a.part_tokens * a.group + (int64_t)t * a.group + tile0 + r;
      *reinterpret_cast<v4f*>(a.part_o + at * a.dim + 4 * d4) = y;
      if (d4 == 0) *reinterpret_cast<v2f*>(a.part_ml + at * 2) = v2f{mx, sum};
    }
  }
}

// Workgroups that a launch of scores aims at. 512 / 768 / 1,024 / 2,048, us of scores and choice, 512 rows of 4 kv heads of 8 f16 heads of 64, 128, 256
// and 512 pages: 36 / 34 / 33 / 33, 41.7 / 39.1 / 37.9 / 40.4, 58 / 56 / 57 / 60; 2,048 rows, of 128: 111 / 100 / 94 / 94.
constexpr int64_t kScoreGroups = 1024;
// Rows (of all kv heads) up to which one launch does both, a workgroup a row: one on every CU. More of them leave the choices, a
// wave each, to wait for each other; few of them on many pages leave CUs idle that could read bounds. One launch against two, us, 32 / 8 bf16 heads
// of 128: 64 pages, 8 / 64 / 256 / 512 / 1,024 rows: 8.8 against 13.0, 9.7 / 13.8, 10.1 / 14.3, 16.4 / 15.5, 29.8 / 18.0; 256 pages, 8 / 64 / 256 /
// 512 rows: 12.2 / 13.7, 13.3 / 15.0, 13.2 / 18.6, 24.7 / 24.8; 512 pages, 8 / 64 / 128 / 256 / 512 rows: 15.8 / 13.6, 16.1 / 15.7, 16.9 / 19.1, 19.0 /
// 25.7, 34.0 / 35.7. Rows of one sequence share what two launches read: 64 rows of two sequences on 64 pages 9.7 / 13.5, 128 of one on 512 17.3 / 18.5.
// The one limit for all numbers of pages costs 2 us at 512 rows of 512 pages. kPickPages ends the rule, and with it the choice by one wave: 8 intervals
// a lane. Beyond, a row takes 16 waves, and 8 / 64 / 256 / 512 rows of 512, 513, 683 and 1,024 pages take 13 / 15 / 19 / 36, 22 / 24 / 33 / 58, 21 / 25 /
// 37 / 65 and 21 / 27 / 43 / 77 us: a step of 8 to 22 us at 513 pages.
constexpr int64_t kPickRows = 256;

// lanes that hold a head's values, 8 each: their number's logarithm
int lanes_log2(int dim) {
  int log2 = 0;
  while ((8 << log2) < dim) ++log2;
  return log2;
}

}  // namespace

hipError_t launch_page_bounds(int cache_type, const AttnArgs& a, const int32_t* from, int64_t slots, uint16_t* bounds,
                              hipStream_t s) {
  const int64_t items = a.batch * slots * a.cache.kv_heads, most = (int64_t)1 << 25;  // (2^31 threads a launch)
  for (int64_t i = 0; i < items; i += most) {
    const dim3 grid((uint32_t)(((items - i < most ? items - i : most) + 3) / 4));
    if (cache_type == DQ_F16)
      hipLaunchKernelGGL((k_page_bounds<DQ_F16>), grid, dim3(256), 0, s, a, from, slots, bounds, lanes_log2(a.dim), i, items);
    else
      hipLaunchKernelGGL((k_page_bounds<DQ_BF16>), grid, dim3(256), 0, s, a, from, slots, bounds, lanes_log2(a.dim), i, items);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_choose_pages(int type, int cache_type, const AttnArgs& a, const ChooseArgs& c, hipStream_t s) {
  int rows_log2 = 0;
  while ((1 << rows_log2) < a.group && rows_log2 < 4) ++rows_log2;
  const int slots = 16 >> rows_log2;
  for (int64_t t = 0; t < a.tokens; t += c.tokens) {
    const int64_t rows = (a.tokens - t < c.tokens ? a.tokens - t : c.tokens) * a.cache.kv_heads;
    const hipError_t e = by_types(type, cache_type, [&](auto tq, auto tc) {
      const int log2 = lanes_log2(a.dim);
      if (c.pages > c.count && rows <= kPickRows && (c.pages <= kPickPages / 2 || (c.pages <= kPickPages && rows >= kPickRows / 2))) {
        const dim3 grid((uint32_t)rows);
        if (a.dim <= 64)
          hipLaunchKernelGGL((k_page_pick<tq(), tc(), 64>), grid, dim3(1024), 0, s, a, c, (int)t, log2);
        else if (a.dim <= 128)
          hipLaunchKernelGGL((k_page_pick<tq(), tc(), 128>), grid, dim3(1024), 0, s, a, c, (int)t, log2);
        else
          hipLaunchKernelGGL((k_page_pick<tq(), tc(), 256>), grid, dim3(512), 0, s, a, c, (int)t, log2);
        return hipGetLastError();
      }
      if (c.pages > c.count) {  // (else every page is read)
        const int64_t tiles = (a.max_q + slots - 1) / slots, groups = (int64_t)a.batch * a.cache.kv_heads * ((c.pages + 63) / 64);
        const int64_t ranges = std::max<int64_t>(1, std::min(tiles, kScoreGroups / groups)), per = (tiles + ranges - 1) / ranges * slots;
        const dim3 grid((uint32_t)(groups * ranges));
        if (a.dim <= 64)
          hipLaunchKernelGGL((k_page_scores<tq(), tc(), 64>), grid, dim3(256), 0, s, a, c, (int)t, rows_log2, (int)ranges, (int)per);
        else if (a.dim <= 128)
          hipLaunchKernelGGL((k_page_scores<tq(), tc(), 128>), grid, dim3(256), 0, s, a, c, (int)t, rows_log2, (int)ranges, (int)per);
        else
          hipLaunchKernelGGL((k_page_scores<tq(), tc(), 256>), grid, dim3(256), 0, s, a, c, (int)t, rows_log2, (int)ranges, (int)per);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
      }
      if (c.pages <= 8 * 64)
        hipLaunchKernelGGL((k_page_choice<tq(), tc(), 8, 1, true>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s, a, c, (int)t, rows, log2);
      else if (c.pages <= 8 * 16 * 64)
        hipLaunchKernelGGL((k_page_choice<tq(), tc(), 8, 16, true>), dim3((uint32_t)rows), dim3(1024), 0, s, a, c, (int)t, rows, log2);
      else
        hipLaunchKernelGGL((k_page_choice<tq(), tc(), 1, 16, false>), dim3((uint32_t)rows), dim3(1024), 0, s, a, c, (int)t, rows, log2);
      return hipGetLastError();
    });
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_page_attention(int type, int cache_type, const AttnArgs& a, const int32_t* chosen, int64_t count,
                                 int32_t splits, int32_t chunk, hipStream_t s) {
  const int tiles = (a.group + 15) / 16;
  const dim3 grid((uint32_t)((int64_t)a.tokens * a.cache.kv_heads * tiles * splits));
  const hipError_t e = by_types(type, cache_type, [&](auto tq, auto tc) {
    if (a.dim <= 64)
      hipLaunchKernelGGL((k_page_attn<tq(), tc(), 64>), grid, dim3(256), 0, s, a, chosen, count, splits, chunk, tiles);
    else if (a.dim <= 128)
      hipLaunchKernelGGL((k_page_attn<tq(), tc(), 128>), grid, dim3(256), 0, s, a, chosen, count, splits, chunk, tiles);
    else
      hipLaunchKernelGGL((k_page_attn<tq(), tc(), 256>), grid, dim3(256), 0, s, a, chosen, count, splits, chunk, tiles);
    return hipGetLastError();
  });
  if (e != hipSuccess || a.part_o == nullptr) return e;
  return launch_join(type, cache_type, a, splits, s);
}

}  // namespace dq
