// dq_pages.hip -- the pages that a query reads: each page's bounds of its keys' channels, the choice of pages
// by an upper bound of a row's scores on them, and attention over the chosen pages alone.
#include <type_traits>

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

// ---- bounds of a page -------------------------------------------------------
// A wave takes a page of a kv head: a lane 8 channels of every 64 / lanes'th key. 16-bit floats are compared as
// whole numbers of their order (negative ones with their other bits turned round), two at a time; NaN lies
// beyond the infinities there, at either end.

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
// Scores decide which pages are read, so two that differ must not tie for a rounding: sums are 64 bits wide
// (products of 16 or 24-bit values are exact in them). They go to the workspace as whole numbers that
// order as they do.

constexpr uint64_t kAlways = ~0ull, kNanKey = ~0ull - 1;

DQ_DEV uint64_t order_key(double x) {
  if (x != x) return kNanKey;
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);  // (-0 is 0)
  return b >> 63 ? ~b : b | 1ull << 63;
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

// A wave scores kRun pages of a row's kv head: 64 / lanes of them at a time, a lane 8 channels of one.
constexpr int kRun = 64;

template <int T, int TC>
__global__ __launch_bounds__(256) void k_page_scores(AttnArgs a, ChooseArgs c, int64_t token0, int lanes_log2, int64_t items) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (item >= items) return;
  const int runs = (c.pages + kRun - 1) / kRun, hk = a.cache.kv_heads;
  const int run = (int)(item % runs), h = (int)(item / runs % hk);
  const int64_t row = item / runs / hk;
  const int t = (int)(token0 + row);
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  const int pages = (row_sees(a, b, t, seq_len(a, b)) + a.cache.page_size - 1) / a.cache.page_size;
  if (run * kRun >= pages) return;
  const int32_t* list = a.pages + b * a.pages_stride;
  const int lanes = 1 << lanes_log2, step = 64 >> lanes_log2, d = 8 * (lane & (lanes - 1));
  const bool in = d < a.dim;
  uint64_t* out = c.keys + (row * hk + h) * c.pages;
  const int end = min(pages, (run + 1) * kRun);
  for (int p0 = run * kRun; p0 < end; p0 += 2 * step) {
    v4u lo[2], hi[2];
    int id[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int p = min(p0 + u * step + (lane >> lanes_log2), end - 1);
      id[u] = list[p];
      const bool ok = (u32)id[u] < (u32)a.cache.n_pages;
      const uint16_t* x = c.bounds + ((int64_t)(ok ? id[u] : 0) * hk + h) * 2 * a.dim + (in ? d : 0);
      lo[u] = *reinterpret_cast<const v4u*>(x);
      hi[u] = *reinterpret_cast<const v4u*>(x + a.dim);
      id[u] = ok;
    }
    uint64_t best[2] = {0, 0};
    for (int i = 0; i < a.group; ++i) {
      const int64_t at = (int64_t)t * a.q_token + (int64_t)(h * a.group + i) * a.q_head + d;
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = in ? load1<T>(a.q, at + e) : 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        double s = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const u32 x = q[e] > 0 ? hi[u][e / 2] : lo[u][e / 2];
          s = fma((double)q[e], (double)(e % 2 ? widen_hi<TC>(x) : widen<TC>(x)), s);
        }
        s = lanes_sum(in ? s : 0.0, lanes_log2);
        const uint64_t key = order_key(s);
        best[u] = key > best[u] ? key : best[u];
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int p = p0 + u * step + (lane >> lanes_log2);
      if (p < end && (lane & (lanes - 1)) == 0) out[p] = id[u] ? best[u] : kNanKey;
    }
  }
}

// The choice: a wave takes a row's kv head, and finds the count-th largest key bit by bit.
// kHeld: all of a row's keys lie in registers, N to a lane; else they are read again for every bit.
template <int N, bool kHeld>
__global__ __launch_bounds__(256) void k_page_choice(AttnArgs a, ChooseArgs c, int64_t token0, int64_t rows) {
  const int lane = threadIdx.x & 63, hk = a.cache.kv_heads;
  const int64_t row = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (row >= rows) return;
  const int t = (int)(token0 + row / hk);
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  const int pages = (row_sees(a, b, t, seq_len(a, b)) + a.cache.page_size - 1) / a.cache.page_size;
  int32_t* out = c.chosen + ((int64_t)t * hk + row % hk) * c.count;
  const int count = (int)min(c.count, (int64_t)pages);
  for (int64_t i = count + lane; i < c.count; i += 64) out[i] = -1;
  if (pages <= c.count) {
    for (int i = lane; i < pages; i += 64) out[i] = i;
    return;
  }
  const uint64_t* keys = c.keys + row * c.pages;
  auto key_at = [&](int p) {
    if (p >= pages) return (uint64_t)0;  // (below every score)
    return p < c.first || p >= pages - c.last ? kAlways : keys[p];
  };
  uint64_t k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = kHeld ? key_at(i * 64 + lane) : 0;
  const int rounds = kHeld ? N : (pages + 63) / 64;
  uint64_t least = 0;
  int taken = 0;  // keys >= least, once they are `count`
#pragma unroll 1
  for (int bit = 63; bit >= 0 && taken != count; --bit) {
    const uint64_t mid = least | 1ull << bit;
    int n = 0;
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < N; ++i) n += __popcll(__ballot(k[i] >= mid));
    } else {
      for (int i = 0; i < rounds; ++i) n += __popcll(__ballot(key_at(i * 64 + lane) >= mid));
    }
    if (n >= count) {
      least = mid;
      taken = n;
    }
  }
  // those above `least`, and of those at it the first ones
  int above = 0;
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < N; ++i) above += __popcll(__ballot(k[i] > least));
  } else {
    for (int i = 0; i < rounds; ++i) above += __popcll(__ballot(key_at(i * 64 + lane) > least));
  }
  int equal = count - above, at = 0;
  auto put = [&](int i, uint64_t key) {
    const uint64_t before = (1ull << lane) - 1, ties = __ballot(key == least);
    const bool mine = key > least || (key == least && __popcll(ties & before) < equal);
    const uint64_t all = __ballot(mine);
    if (mine) out[at + __popcll(all & before)] = i * 64 + lane;
    at += __popcll(all);
    equal -= min(equal, __popcll(ties));
  };
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < N; ++i) put(i, k[i]);
  } else {
    for (int i = 0; i < rounds; ++i) put(i, key_at(i * 64 + lane));
  }
}

// ---- attention over chosen pages ---------------------------------------------
// An item is (token, kv head, up to 16 of its query heads, range of the list): its rows see the same keys. The four
// waves take 32 keys each in turn, with a running softmax of their own, and add up at the end. Scores are S^T = K
// Q^T, which leaves a lane with the weights that O^T = V^T P^T takes from it; keys and values go straight
// from memory to registers (a lane's 16 bytes of a key are its A operand, of the values it takes DP / 16 of 8 keys).

template <int DP>
struct PageLds {
  v4f o[4][16][DP / 4];
  float ml[4][16][2];
  int bad;
};

template <int DP>
struct PageKv {
  v4u k[2][DP / 32];
  u32 v[8][DP / 32];
};

// Moves x of the lanes in `mask` to lanes 0, 1, ... in turn.
DQ_DEV int to_front(int x, uint64_t mask, int lane) {
  const uint64_t before = (1ull << lane) - 1;
  const int to = mask >> lane & 1 ? __popcll(mask & before) : __popcll(mask) + __popcll(~mask & before);
  return __builtin_amdgcn_ds_permute(4 * to, x);
}

template <int T, int TC, int DP>
__global__ __launch_bounds__(256) void k_page_attn(AttnArgs a, const int32_t* chosen, int64_t count, int splits, int chunk, int tiles) {
  constexpr int NP = kParts<T, TC>;
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
  const int b = find_seq(a, t, lane);
  if (b < 0) return;
  if (threadIdx.x == 0) sh.bad = 0;
  __syncthreads();
  const int rows = min(16, a.group - tile0);
  const int sees = row_sees(a, b, t, seq_len(a, b));
  RawQ<T, DP> raw;
  load_q<T, DP>(a, n < rows, t, head * a.group + tile0 + min(n, rows - 1), g, raw);
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
  u32 koff[DP / 32], voff[DP / 128 > 0 ? DP / 128 : 1];
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) koff[s] = 32 * s + 8 * g < a.dim ? n * token_bytes + (32 * s + 8 * g) * 2 : kOut;
#pragma unroll
  for (int s = 0; s < (DP / 128 > 0 ? DP / 128 : 1); ++s) {
    const int d = n * NC + 8 * s;
    voff[s] = d < a.dim ? 4 * g * token_bytes + d * 2 : kOut;
  }

  const int units = ca.page_size / 16;  // of 16 keys, of a page
  const int skip = 8 / units, skip_rest = 8 % units;
  const int64_t e0 = (int64_t)range * chunk, e1 = min(e0 + chunk, count);
  const int32_t* list = chosen + ((int64_t)t * ca.kv_heads + head) * count;
  for (int64_t eb = e0; eb < e1; eb += 64) {
    // the next 64 entries, a lane each; those that hold visible keys to the front
    int entry = eb + lane < e1 ? list[eb + lane] : -1;
    const bool some = entry >= 0 && (int64_t)entry * ca.page_size < sees;
    int id = some ? a.pages[b * a.pages_stride + entry] : 0;
    if ((u32)id >= (u32)ca.n_pages) {
      bad = true;
      id = 0;
    }
    const uint64_t mask = __ballot(some);
    entry = to_front(entry, mask, lane);
    id = to_front(id, mask, lane);
    const int halves = __popcll(mask) * units;  // of tiles: runs of 16 keys
    int e = 2 * wave / units, sub = 2 * wave % units;
    for (int half = 2 * wave; half < halves; half += 8) {
      PageKv<DP> r;
      int kb[2];
      int64_t base[2];
      {
        const int id0 = __builtin_amdgcn_readlane(id, e);
        kb[0] = __builtin_amdgcn_readlane(entry, e) * ca.page_size + 16 * sub;
        base[0] = id0 * ca.page + 16 * sub * ca.token + head * ca.head;
        kb[1] = INT32_MAX - 16;  // (no key)
        base[1] = base[0];
        if (half + 1 < halves) {
          const bool over = sub + 1 == units;
          const int e2 = over ? e + 1 : e, sub2 = over ? 0 : sub + 1;
          kb[1] = __builtin_amdgcn_readlane(entry, e2) * ca.page_size + 16 * sub2;
          base[1] = __builtin_amdgcn_readlane(id, e2) * ca.page + 16 * sub2 * ca.token + head * ca.head;
        }
        e += skip;
        sub += skip_rest;
        if (sub >= units) {
          sub -= units;
          ++e;
        }
      }
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const auto kr = rsrc(ca.k + base[t2], 0x7FFFFFFFu);
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) r.k[t2][s] = ld16(kr, koff[s]);
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
      float x[8];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        v4f acc = {0, 0, 0, 0};
#pragma unroll
        for (int p = NP - 1; p >= 0; --p)
#pragma unroll
          for (int s = 0; s < DP / 32; ++s) acc = mma<TC>(r.k[t2][s], q[p][s], acc);
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
        for (int w = 0; w < 4; ++w)
          vt[w] = __builtin_amdgcn_perm(r.v[2 * w + 1][i >> 1], r.v[2 * w][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) o[i] = mma<TC>(vt, p[k], o[i]);
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
    for (int w = 0; w < NC / 4; ++w) sh.o[wave][n][d / 4 + w] = v4f{o[4 * w][i], o[4 * w + 1][i], o[4 * w + 2][i], o[4 * w + 3][i]};
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
      y += sh.o[k][r][d4] * f;
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
  const int64_t runs = (c.pages + kRun - 1) / kRun;
  for (int64_t t = 0; t < a.tokens; t += c.tokens) {
    const int64_t rows = (a.tokens - t < c.tokens ? a.tokens - t : c.tokens) * a.cache.kv_heads, items = rows * runs;
    if (c.pages > c.count) {  // (else every page is read)
      const hipError_t e = by_types(type, cache_type, [&](auto tq, auto tc) {
        hipLaunchKernelGGL((k_page_scores<tq(), tc()>), dim3((uint32_t)((items + 3) / 4)), dim3(256), 0, s, a, c, t,
                           lanes_log2(a.dim), items);
        return hipGetLastError();
      });
      if (e != hipSuccess) return e;
    }
    const dim3 grid((uint32_t)((rows + 3) / 4));
    if (c.pages <= 8 * 64)
      hipLaunchKernelGGL((k_page_choice<8, true>), grid, dim3(256), 0, s, a, c, t, rows);
    else if (c.pages <= 32 * 64)
      hipLaunchKernelGGL((k_page_choice<32, true>), grid, dim3(256), 0, s, a, c, t, rows);
    else
      hipLaunchKernelGGL((k_page_choice<1, false>), grid, dim3(256), 0, s, a, c, t, rows);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
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
