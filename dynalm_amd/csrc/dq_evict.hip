// dq_evict.hip -- what a cache keeps: the attention weight that each key gathers, the choice of the keys
// that stay, and their move to the front.
#include <algorithm>
#include <cfloat>

#include "dq_attn_device.h"
#include "dq_pages.h"

namespace dq {
namespace {

// A sequence's rows [first, first + n) of all, whatever its offsets hold.
DQ_DEV void seq_rows(const AttnArgs& a, int b, int& first, int& n) {
  const int lo = a.q_offsets != nullptr ? a.q_offsets[b] : b, hi = a.q_offsets != nullptr ? a.q_offsets[b + 1] : b + 1;
  first = min(max(lo, 0), a.tokens);
  n = min(min(max(hi, first), a.tokens) - first, a.max_q);
}

// ---- attention weight ---------------------------------------------------------
// m_j = sum over rows of 2^(c s_rj - z_r), with c = scale log2 e and z_r = lse_r log2 e: S = Q K^T on the matrix
// cores leaves a lane with one key's products with four rows, so that sums over rows stay in their lane until
// the last. z is split in a float and a rest, whose power of two is the factor that a row's weights are added with.

constexpr int kMassTiles = 4;                       // of 16 keys: a wave's
constexpr int kMassKeys = 4 * 16 * kMassTiles;      // a workgroup's

template <int T, int TC, int DP>
__global__ __launch_bounds__(256) void k_mass(AttnArgs a, MassArgs m, int key_tiles) {
  constexpr int NP = kParts<T, TC>;
  const CacheArgs& ca = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  u32 item = blockIdx.x;
  const int head = item % ca.kv_heads;
  item /= ca.kv_heads;
  const int kt = item % key_tiles;
  item /= key_tiles;
  const int range = item % m.splits, b = item / m.splits;
  const int len = seq_len(a, b), k0 = (kt * 4 + wave) * 16 * kMassTiles;
  if (k0 >= len) return;
  int first, count;
  seq_rows(a, b, first, count);
  const int old = len - count;  // keys before the rows' own

  // the wave's keys as B operands: lane n of a group has key n, 8 (lane / 16) .. + 7 of every 32 values
  v4u k[kMassTiles][DP / 32];
  bool bad[kMassTiles];
  const int32_t* list = a.pages + b * a.pages_stride;
  const u32 token_bytes = (u32)ca.token * 2;
#pragma unroll
  for (int i = 0; i < kMassTiles; ++i) {
    const int key = k0 + 16 * i, p = min(key, len - 1) / ca.page_size;
    int id = page_at(list, p);
    bad[i] = (u32)id >= (u32)ca.n_pages;
    if (bad[i]) id = 0;
    const int in = key < len ? key - p * ca.page_size : 0;
    const auto kr = rsrc(ca.k + id * ca.page + in * ca.token + head * ca.head, 0x7FFFFFFFu);
#pragma unroll
    for (int s = 0; s < DP / 32; ++s)
      k[i][s] = ld16(kr, key < len && 32 * s + 8 * g < a.dim ? n * token_bytes + (32 * s + 8 * g) * 2 : 0x80000000u);
  }

  float sum[kMassTiles];
#pragma unroll
  for (int i = 0; i < kMassTiles; ++i) sum[i] = 0;
  // rows before the first that sees key k0 add nothing
  const int rows = count * a.group;
  const int64_t sees_from = max((int64_t)0, (int64_t)(k0 - old) * a.group);
  const int r_end = (int)min((int64_t)rows, m.splits > 1 ? (int64_t)(range + 1) * m.rows : (int64_t)rows);
  int r0 = (int)max((int64_t)range * m.rows, sees_from / 16 * 16);
  for (; r0 < r_end; r0 += 16) {
    const int r = min(r0 + n, rows - 1), token = first + r / a.group, qh = head * a.group + r % a.group;
    const bool valid = r0 + n < r_end;
    RawQ<T, DP> raw;
    load_q<T, DP>(a, valid, token, qh, g, raw);
    const float lse = m.lse[(int64_t)token * a.heads + qh];
    v4u q[NP][DP / 32];
    const float c = q_operands<T, TC, DP>(a, raw, q);
    const double z = (double)lse * 1.4426950408889634074;
    float hi = (float)z, f = exp2_fast((float)((double)hi - z));
    int limit = valid ? old + (token - first) + 1 : 0;
    if (fabsf(hi) == INFINITY) {
      hi = fabsf(lse) == INFINITY ? INFINITY : copysignf(FLT_MAX, lse);  // (a row whose lse is -inf has no weights)
      f = 1.f;
    }
    // of the four rows whose products the lane holds
    float c4[4], hi4[4], f4[4];
    int limit4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c4[i] = T == DQ_F32 ? __shfl(c, 4 * g + i, 64) : c;
      hi4[i] = __shfl(hi, 4 * g + i, 64);
      f4[i] = __shfl(f, 4 * g + i, 64);
      limit4[i] = __shfl(limit, 4 * g + i, 64);
    }
#pragma unroll
    for (int i = 0; i < kMassTiles; ++i) {
      v4f acc = {0, 0, 0, 0};
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) acc = mma<TC>(q[p][s], k[i][s], acc);
      const int key = k0 + 16 * i + n;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = exp2_fast(fmaf(acc[e], c4[e], -hi4[e])) * f4[e];
        sum[i] += key < limit4[e] ? w : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMassTiles; ++i) sum[i] = row_sum(sum[i]);
  // lane group i writes tile i
  static_assert(kMassTiles == 4);
  float x = g == 0 ? sum[0] : g == 1 ? sum[1] : g == 2 ? sum[2] : sum[3];
  if (g == 0 ? bad[0] : g == 1 ? bad[1] : g == 2 ? bad[2] : bad[3]) x = __builtin_nanf("");
  const int key = k0 + 16 * g + n;
  if (key >= len) return;
  if (m.part != nullptr) {
    m.part[(((int64_t)range * a.batch + b) * ca.kv_heads + head) * a.max_len + key] = x;
    return;
  }
  float* out = m.mass + b * m.seq + head * m.head + key;
  *out = m.decay != 0 && key < old ? fmaf(m.decay, *out, x) : x;
}

// Adds the ranges of rows that were summed apart.
__global__ __launch_bounds__(256) void k_mass_join(AttnArgs a, MassArgs m, int64_t keys) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= keys) return;
  const int key = (int)(at % a.max_len), head = (int)(at / a.max_len % a.cache.kv_heads), b = (int)(at / a.max_len / a.cache.kv_heads);
  const int len = seq_len(a, b);
  if (key >= len) return;
  int first, count;
  seq_rows(a, b, first, count);
  float x = 0;
  for (int s = 0; s < m.splits; ++s) x += m.part[s * keys + at];
  float* out = m.mass + b * m.seq + head * m.head + key;
  *out = m.decay != 0 && key < len - count ? fmaf(m.decay, *out, x) : x;
}

// ---- the keys that stay ---------------------------------------------------------
// A workgroup takes a sequence's kv head and finds the budget-th largest weight bit by bit, of whole numbers that
// order as the weights do. Wave w holds (or, kHeld false, reads again for each bit) a run of the places, so that the list comes out ascending.

constexpr int kKeepWaves = 16;

// (NaN 1, below all numbers; -inf 0x7FFFFF, +inf 0xFF800000; 0 is no key's)
DQ_DEV u32 weight_key(float x) {
  const u32 b = as_u(x + 0.f);  // (-0 is 0)
  if (x != x) return 1;
  return b >> 31 ? ~b : b | 0x80000000u;
}

template <int N, bool kHeld>
__global__ __launch_bounds__(kKeepWaves * 64) void k_keep(KeepArgs a) {
  __shared__ int counts[2][kKeepWaves], ties[kKeepWaves];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int h = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads;
  const int len = a.max_len > 0 ? min(max(a.lens[b], 0), a.max_len) : 0;
  const int budget = (int)min(a.budget, (int64_t)len);
  int32_t* out = a.kept + ((int64_t)b * a.kv_heads + h) * a.budget;
  if (threadIdx.x == 0 && h == 0 && a.kept_lens != nullptr) a.kept_lens[b] = budget;
  for (int64_t i = budget + (int)threadIdx.x; i < a.budget; i += kKeepWaves * 64) out[i] = -1;
  if (len <= a.budget) {
    for (int i = threadIdx.x; i < len; i += kKeepWaves * 64) out[i] = i;
    return;
  }
  const float* mass = a.mass + b * a.seq + h * a.head;
  const int rounds = kHeld ? N : (len + kKeepWaves * 64 - 1) / (kKeepWaves * 64);
  const int64_t base = (int64_t)wave * 64 * rounds;
  auto key_at = [&](int i) -> u32 {
    const int64_t p = base + i * 64 + lane;
    if (p >= len) return 0;
    return p < a.first || p >= len - a.last ? 0xFFFFFFFFu : weight_key(mass[p]);
  };
  u32 k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = kHeld ? key_at(i) : 0;
  auto count_if = [&](auto&& f) {
    int n = 0;
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < N; ++i) n += __popcll(__ballot(f(k[i])));
    } else {
      for (int i = 0; i < rounds; ++i) n += __popcll(__ballot(f(key_at(i))));
    }
    return n;
  };
  u32 least = 0;
  int taken = 0, turn = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0 && taken != budget; --bit, turn ^= 1) {
    const u32 mid = least | 1u << bit;
    const int mine = count_if([&](u32 x) { return x >= mid; });
    if (lane == 0) counts[turn][wave] = mine;
    __syncthreads();  // (the other turn's counts are read before it, written after the next)
    int n = 0;
#pragma unroll
    for (int w = 0; w < kKeepWaves; ++w) n += counts[turn][w];
    if (n >= budget) {
      least = mid;
      taken = n;
    }
  }
  const int above = count_if([&](u32 x) { return x > least; }), equal = count_if([&](u32 x) { return x == least; });
  __syncthreads();
  if (lane == 0) {
    counts[0][wave] = above;
    ties[wave] = equal;
  }
  __syncthreads();
  int all_above = 0, above_before = 0, ties_before = 0;
#pragma unroll
  for (int w = 0; w < kKeepWaves; ++w) {
    all_above += counts[0][w];
    if (w < wave) {
      above_before += counts[0][w];
      ties_before += ties[w];
    }
  }
  const int room = budget - all_above;  // for keys at `least`, the first ones
  int left = max(room - ties_before, 0), at = above_before + min(ties_before, room);
  auto put = [&](int i, u32 x) {
    const uint64_t before = (1ull << lane) - 1, tie = __ballot(x == least);
    const bool mine = x > least || (x == least && __popcll(tie & before) < left);
    const uint64_t all = __ballot(mine);
    if (mine) out[at + __popcll(all & before)] = (int)(base + i * 64 + lane);
    at += __popcll(all);
    left -= min(left, __popcll(tie));
  };
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < N; ++i) put(i, k[i]);
  } else {
    for (int i = 0; i < rounds; ++i) put(i, key_at(i));
  }
}

// ---- their move ------------------------------------------------------------------
// A workgroup takes a run of the keys, or of the values, of a sequence's kv head. In place it takes all of them, one
// run after the other: a run is read whole before it is written, and places that ascend lie at their number or behind it,
// so that later runs read nothing that was written. The weights, which may be moved in place beside keys that are not,
// are always one workgroup's.

constexpr int kMoveLoads = 8;  // of 16 bytes (a weight), a thread's of a run

// All reads of the workgroup have come.
DQ_DEV void reads_done() {
  wait_loads();
  __syncthreads();
}

DQ_DEV void move_weights(const int32_t* kept, int64_t count, int len, const float* mass, float* out) {
  for (int64_t i0 = 0; i0 < count; i0 += 256 * kMoveLoads) {
    float w[kMoveLoads];
    bool moves[kMoveLoads];
#pragma unroll
    for (int u = 0; u < kMoveLoads; ++u) {
      const int64_t i = i0 + u * 256 + threadIdx.x;
      const int place = i < count ? kept[i] : -1;
      moves[u] = place >= 0 && place < len;
      w[u] = moves[u] ? mass[place] : 0.f;
    }
    reads_done();
#pragma unroll
    for (int u = 0; u < kMoveLoads; ++u)
      if (moves[u]) out[i0 + u * 256 + threadIdx.x] = w[u];
  }
}

template <bool kInPlace>
__global__ __launch_bounds__(256) void k_compact(AttnArgs a, CompactArgs c, int lanes_log2, int runs) {
  const CacheArgs& ca = a.cache;
  const int jobs = 2 * (kInPlace ? 1 : runs) + (c.mass != nullptr);
  u32 item = blockIdx.x;
  const int h = item % ca.kv_heads;
  item /= ca.kv_heads;
  const int job = item % jobs, b = item / jobs;
  const int len = seq_len(a, b);
  const int32_t* kept = c.kept + ((int64_t)b * ca.kv_heads + h) * c.budget;
  const int64_t most = min(c.budget, (int64_t)len);  // (entries behind are none of kv_keep's)
  if (c.mass != nullptr && job == jobs - 1) {
    const int64_t at = b * c.seq + h * c.head;
    move_weights(kept, most, len, c.mass + at, c.mass_out + at);
    return;
  }
  const int32_t* from = a.pages + b * a.pages_stride;
  const int32_t* to = kInPlace ? from : c.to_pages + b * c.to_stride;
  uint16_t* pool = (job & 1 ? ca.v : ca.k) + h * ca.head;
  const int rows = 256 >> lanes_log2, r = threadIdx.x >> lanes_log2, d = 8 * (threadIdx.x & ((1 << lanes_log2) - 1));
  const int run_rows = rows * kMoveLoads, run0 = kInPlace ? 0 : job >> 1;
  for (int run = run0; run < (kInPlace ? runs : run0 + 1); ++run) {
    const int64_t i0 = (int64_t)run * run_rows;
    if (i0 >= most) break;  // (all threads)
    v4u x[kMoveLoads];
    int64_t target[kMoveLoads];
#pragma unroll
    for (int u = 0; u < kMoveLoads; ++u) {
      const int64_t i = i0 + u * rows + r;
      const int place = i < most && d < a.dim ? kept[i] : -1;
      target[u] = -1;
      if (place < 0 || place >= len) continue;
      const int sp = place / ca.page_size, tp = (int)i / ca.page_size;
      const int sid = from[sp], tid = to[tp];
      if ((u32)sid >= (u32)ca.n_pages || (u32)tid >= (u32)ca.n_pages) continue;
      x[u] = *reinterpret_cast<const v4u*>(pool + sid * ca.page + (place - sp * ca.page_size) * ca.token + d);
      target[u] = tid * ca.page + ((int)i - tp * ca.page_size) * ca.token + d;
    }
    if (kInPlace) reads_done();
#pragma unroll
    for (int u = 0; u < kMoveLoads; ++u)
      if (target[u] >= 0) *reinterpret_cast<v4u*>(pool + target[u]) = x[u];
  }
}

}  // namespace

hipError_t launch_attention_mass(int type, int cache_type, const AttnArgs& a, const MassArgs& m, hipStream_t s) {
  const int tiles = (a.max_len + kMassKeys - 1) / kMassKeys;
  const dim3 grid((uint32_t)((int64_t)a.batch * m.splits * tiles * a.cache.kv_heads));
  const hipError_t e = by_types(type, cache_type, [&](auto tq, auto tc) {
    if (a.dim <= 64)
      hipLaunchKernelGGL((k_mass<tq(), tc(), 64>), grid, dim3(256), 0, s, a, m, tiles);
    else if (a.dim <= 128)
      hipLaunchKernelGGL((k_mass<tq(), tc(), 128>), grid, dim3(256), 0, s, a, m, tiles);
    else
      hipLaunchKernelGGL((k_mass<tq(), tc(), 256>), grid, dim3(256), 0, s, a, m, tiles);
    return hipGetLastError();
  });
  if (e != hipSuccess || m.part == nullptr) return e;
  const int64_t keys = (int64_t)a.batch * a.cache.kv_heads * a.max_len;
  hipLaunchKernelGGL(k_mass_join, dim3((uint32_t)((keys + 255) / 256)), dim3(256), 0, s, a, m, keys);
  return hipGetLastError();
}

hipError_t launch_kv_keep(int64_t batch, const KeepArgs& k, hipStream_t s) {
  const dim3 grid((uint32_t)(batch * k.kv_heads)), block(kKeepWaves * 64);
  constexpr int kLanes = kKeepWaves * 64;
  if (k.max_len <= 4 * kLanes)
    hipLaunchKernelGGL((k_keep<4, true>), grid, block, 0, s, k);
  else if (k.max_len <= 16 * kLanes)
    hipLaunchKernelGGL((k_keep<16, true>), grid, block, 0, s, k);
  else if (k.max_len <= 64 * kLanes)
    hipLaunchKernelGGL((k_keep<64, true>), grid, block, 0, s, k);
  else
    hipLaunchKernelGGL((k_keep<1, false>), grid, block, 0, s, k);
  return hipGetLastError();
}

hipError_t launch_kv_compact(const AttnArgs& a, const CompactArgs& c, hipStream_t s) {
  int log2 = 0;
  while ((8 << log2) < a.dim) ++log2;
  const int64_t rows = (256 >> log2) * kMoveLoads;
  const int runs = (int)((std::min(c.budget, (int64_t)a.max_len) + rows - 1) / rows);
  const bool in_place = c.to_pages == nullptr;
  const int64_t jobs = 2 * (in_place ? 1 : runs) + (c.mass != nullptr);
  const dim3 grid((uint32_t)(jobs * a.batch * a.cache.kv_heads));
  if (in_place)
    hipLaunchKernelGGL((k_compact<true>), grid, dim3(256), 0, s, a, c, log2, runs);
  else
    hipLaunchKernelGGL((k_compact<false>), grid, dim3(256), 0, s, a, c, log2, runs);
  return hipGetLastError();
}

}  // namespace dq
