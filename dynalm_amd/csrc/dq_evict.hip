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

constexpr int kMassKeys = 256;  // a workgroup's
constexpr int kMassTiles = 4;   // of 16 keys: a wave's, of four

// z = lse log2 e as a float and the power of two of what that leaves out, half a unit of its last place. Past 2^24 that is more than
// 1, and no more than the scores' own rounding there: 1 of it is taken, so that the factor is never 0 or infinite beside a weight that is.
DQ_DEV void split_lse(float lse, float& hi, float& f) {
  const double z = (double)lse * 1.4426950408889634074;
  hi = (float)z;
  f = exp2_fast(__builtin_amdgcn_fmed3f((float)((double)hi - z), -1.f, 1.f));
  if (fabsf(hi) == INFINITY) {
    hi = fabsf(lse) == INFINITY ? INFINITY : copysignf(FLT_MAX, lse);  // (-inf too: such a row has no weights)
    f = 1.f;
  }
}

// A wave's keys as B operands: lane n of a group has key n, 8 (lane / 16) .. + 7 of every 32 values.
template <int DP, int M>
DQ_DEV void load_keys(const AttnArgs& a, int b, int head, int k0, int len, int n, int g, v4u (&k)[M][DP / 32], bool (&bad)[M]) {
  const CacheArgs& ca = a.cache;
  const int32_t* list = a.pages + b * a.pages_stride;
  const u32 token_bytes = (u32)ca.token * 2;
#pragma unroll
  for (int i = 0; i < M; ++i) {
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
}

// The sums over a wave's rows into the weights, or into the range's part.
template <int M>
DQ_DEV void put_mass(const AttnArgs& a, const MassArgs& m, int b, int head, int part, int k0, int len, int old, int n, int g, float (&sum)[M],
                     const bool (&bad)[M]) {
  const CacheArgs& ca = a.cache;
#pragma unroll
  for (int i = 0; i < M; ++i) sum[i] = row_sum(sum[i]);
  // lane group i writes tile i
  static_assert(M == 2 || M == 4);
  float x = g == 0 ? sum[0] : g == 1 ? sum[1] : g == 2 ? sum[M - 2] : sum[M - 1];
  if (g == 0 ? bad[0] : g == 1 ? bad[1] : g == 2 ? bad[M - 2] : bad[M - 1]) x = __builtin_nanf("");
  const int key = k0 + 16 * g + n;
  if (g >= M || key >= len) return;
  if (m.part != nullptr) {
    m.part[(((int64_t)part * a.batch + b) * ca.kv_heads + head) * a.max_len + key] = x;
    return;
  }
  float* out = m.mass + b * m.seq + head * m.head + key;
  *out = m.decay != 0 && key < old ? fmaf(m.decay, *out, x) : x;
}

// Adds the weights of 16 of a sequence's rows (of a kv head: row r is query head r % group of token first + r / group),
// r0 .. up to r_end, on the wave's keys. A row's weight on a key that it does not see is left out, whatever its product; all of
// a row whose lse is -inf are.
template <int T, int TC, int DP, int M>
DQ_DEV void add_rows(const AttnArgs& a, const MassArgs& m, int head, int first, int old, int r0, int r_end, int k0, int n, int g,
                     const v4u (&k)[M][DP / 32], float (&sum)[M]) {
  constexpr int NP = kParts<T, TC>;
  const int r = min(r0 + n, r_end - 1), token = first + r / a.group, qh = head * a.group + r % a.group;
  const bool valid = r0 + n < r_end;
  RawQ<T, DP> raw;
  load_q<T, DP>(a, valid, token, qh, g, raw);
  const float lse = m.lse[(int64_t)token * a.heads + qh];
  v4u q[NP][DP / 32];
  const float c = q_operands<T, TC, DP>(a, raw, q);
  float hi, f;
  split_lse(lse, hi, f);
  const int limit = valid && lse != -INFINITY ? old + (token - first) + 1 : 0;
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
  for (int i = 0; i < M; ++i) {
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

template <int T, int TC, int DP>
__global__ __launch_bounds__(256) void k_mass(AttnArgs a, MassArgs m, int key_tiles) {
  const CacheArgs& ca = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  u32 item = blockIdx.x;
  const int head = item % ca.kv_heads;
  item /= ca.kv_heads;
  const int part = item % m.splits;
  item /= m.splits;
  const int kt = item % key_tiles, b = item / key_tiles;
  const int len = seq_len(a, b), k0 = (kt * 4 + wave) * 16 * kMassTiles;
  if (k0 >= len) return;
  int first, count;
  seq_rows(a, b, first, count);
  const int old = len - count;  // keys before the rows' own

  v4u k[kMassTiles][DP / 32];
  bool bad[kMassTiles];
  load_keys<DP>(a, b, head, k0, len, n, g, k, bad);

  float sum[kMassTiles];
#pragma unroll
  for (int i = 0; i < kMassTiles; ++i) sum[i] = 0;
  // rows before the first that sees key k0 add nothing; of the others every splits-th 16 are this part's
  const int rows = count * a.group;
  const int64_t sees_from = max((int64_t)0, (int64_t)(k0 - old) * a.group);
  for (int64_t at = sees_from + 16 * part; at < rows; at += 16 * m.splits)
    add_rows<T, TC, DP>(a, m, head, first, old, (int)at, rows, k0, n, g, k, sum);
  put_mass(a, m, b, head, part, k0, len, old, n, g, sum, bad);
}

// Many rows: the same with the rows' queries through LDS for all of its waves together, two buffers deep. A tile is as many
// whole tokens as kMassRows rows hold, so that a thread's rows lie at the same offsets from every tile's first token (rows that
// are left have a weight of 0); a row's 16-byte chunks lie at their number XOR some bits of the row's, which spreads a
// column of rows over the banks. The products of 16 rows stand beside the exponentials of the 16 before.
// A prompt of 4,096 tokens, 32 / 8 f16 heads of 128 (68.7 GFLOP, half of the square): 92 us and 6 for the join, 740 TFLOP/s, where a large
// matrix product reaches 1,180. Bound by issue: 16 MFMAs (256 clocks), 16 exponentials (128) and 32 sums (128) of a wave stand for 16 rows x 64 keys;
// the matrix cores are busy 39% of the time, the vector unit 65%. Without the LDS 257 us; with parts that are ranges of rows, not turns, 124 (a
// third of the CUs idle at the end); with a wait for the keys inside the loop 142; four waves a SIMD spill (178).

template <int T>
constexpr int kMassRows = T == DQ_F32 ? 32 : 64;

template <int T, int TC, int DP>
struct MassLds {
  alignas(16) uint16_t q[2][kParts<T, TC>][kMassRows<T> * DP];
  alignas(16) float hi[2][kMassRows<T>], f[2][kMassRows<T>], c[2][kMassRows<T>];
  alignas(16) int token[kMassRows<T>];  // of a tile's row
};

// Waves of a workgroup, for heads over 128 values of 32 keys each, not 64, which with their products leave one wave a SIMD (the
// prompt above in heads of 256: 241 us and 189, with fp32 rows 673 and 449; two workgroups a CU spill, 675).
template <int DP>
constexpr int kMassWaves = DP <= 128 ? 4 : 8;

template <int T, int TC, int DP>
__global__ __launch_bounds__(kMassWaves<DP> * 64) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 3 : 2, DP <= 128 ? 3 : 4))) void k_mass_many(AttnArgs a, MassArgs m, int key_tiles) {
  constexpr int NP = kParts<T, TC>, QR = kMassRows<T>, kBytes = T == DQ_F32 ? 4 : 2;
  constexpr int W = kMassWaves<DP>, M = kMassKeys / 16 / W;
  constexpr int kChunks = DP / 8, kPasses = QR * kChunks / (64 * W), kPassRows = 64 * W / kChunks;
  __shared__ MassLds<T, TC, DP> sh;
  const CacheArgs& ca = a.cache;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  u32 item = blockIdx.x;
  const int head = item % ca.kv_heads;
  item /= ca.kv_heads;
  const int part = item % m.splits;
  item /= m.splits;
  const int kt = item % key_tiles, b = item / key_tiles;  // (the first keys are seen by most rows)
  const int len = seq_len(a, b);
  if (kt * kMassKeys >= len) return;
  const int k0 = kt * kMassKeys + wave * 16 * M;
  int first, count;
  seq_rows(a, b, first, count);
  const int old = len - count;
  const int step = QR / a.group;  // tokens of a tile
  // tokens before the first that sees one of the workgroup's keys add nothing; of the others every splits-th tile is this part's
  const int t_end = first + count, stride = step * m.splits;
  const int t_begin = (int)min((int64_t)t_end, first + max((int64_t)0, (int64_t)kt * kMassKeys - old) + (int64_t)step * part);

  // a thread's 16 bytes (fp32: 32) of a row, kPasses rows of a tile; it is the row's chunk `chunk`
  const int chunk = threadIdx.x % kChunks, pass_row = threadIdx.x / kChunks;
  v4u raw[kPasses][T == DQ_F32 ? 2 : 1];
  u32 off[kPasses], off0[kPasses];  // in bytes from the tile's first token; of the same head of that token
  int tok[kPasses];
  bool in[kPasses];  // (a chunk past the head's values, a row past the tile's tokens is 0)
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = p * kPassRows + pass_row;
    tok[p] = row / a.group;
    in[p] = tok[p] < step && 8 * chunk < a.dim;
    if (!in[p]) tok[p] = 1 << 30;
    off0[p] = in[p] ? (u32)((row % a.group) * (int)a.q_head + 8 * chunk) * kBytes : 0;
    off[p] = off0[p] + (in[p] ? (u32)(tok[p] * (int)a.q_token) * kBytes : 0);
  }
  const int own_row = threadIdx.x % QR, own_token = own_row / a.group;
  if (threadIdx.x < QR) sh.token[own_row] = own_token < step ? own_token : 1 << 30;
  const float* own_lse = m.lse + head * a.group + own_row % a.group;
  float lse = 0;
  bool lse_in = false;
  auto read = [&](int t0) {
    const char* base = static_cast<const char*>(a.q) + ((int64_t)t0 * a.q_token + (int64_t)head * a.group * a.q_head) * kBytes;
    // (a token behind the last: the first; nothing sees it)
    if (a.q_vec) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int k = 0; k < (T == DQ_F32 ? 2 : 1); ++k)
          raw[p][k] = *reinterpret_cast<const v4u*>(base + (t0 + tok[p] < t_end ? off[p] : off0[p]) + 16 * k);
    } else {
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const char* src = base + (t0 + tok[p] < t_end ? off[p] : off0[p]);
#pragma unroll
        for (int i = 0; i < (T == DQ_F32 ? 8 : 4); ++i)
          raw[p][i / 4][i % 4] = T == DQ_F32 ? reinterpret_cast<const u32*>(src)[i]
                                             : (u32)reinterpret_cast<const uint16_t*>(src)[2 * i] | (u32)reinterpret_cast<const uint16_t*>(src)[2 * i + 1] << 16;
      }
    }
    lse_in = own_token < step && t0 + own_token < t_end;
    lse = *(own_lse + ((int64_t)t0 + (lse_in ? own_token : 0)) * a.heads);
  };
  auto place = [&](int row, int ch) { return row * DP + 8 * (ch ^ (DP == 64 ? (row >> 1) & 7 : row & 15)); };
  auto write = [&](int buf) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = p * kPassRows + pass_row;
#pragma unroll
      for (int k = 0; k < (T == DQ_F32 ? 2 : 1); ++k) raw[p][k] = in[p] ? raw[p][k] : v4u{0, 0, 0, 0};
      if constexpr (T != DQ_F32) {
        *reinterpret_cast<v4u*>(&sh.q[buf][0][place(row, chunk)]) = raw[p][0];
      } else {
        // scaled to a largest value in [2^14, 2^15), where all parts are normal numbers
        float most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(as_f(raw[p][i / 4][i % 4])));
#pragma unroll
        for (int s = kChunks / 2; s >= 1; s >>= 1) most = fmaxf(most, __shfl_xor(most, s, 64));
        const int e = most > 0 && most < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
        v4u part[NP];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32 x[NP];
          split<T, TC>(ldexpf(as_f(raw[p][i / 2][i % 2 * 2]), e), ldexpf(as_f(raw[p][i / 2][i % 2 * 2 + 1]), e), x);
#pragma unroll
          for (int k = 0; k < NP; ++k) part[k][i] = x[k];
        }
#pragma unroll
        for (int k = 0; k < NP; ++k) *reinterpret_cast<v4u*>(&sh.q[buf][k][place(row, chunk)]) = part[k];
        if (chunk == 0) sh.c[buf][row] = fmaxf(ldexpf(a.scale_log2, -e), 1.2e-38f);
      }
    }
    if (threadIdx.x < QR) {
      float hi, f;
      split_lse(lse_in ? lse : -INFINITY, hi, f);
      sh.hi[buf][own_row] = hi;
      sh.f[buf][own_row] = f;
    }
  };

  if (t_begin < t_end) read(t_begin);
  v4u k[M][DP / 32];
  bool bad[M];
  load_keys<DP>(a, b, head, k0, len, n, g, k, bad);
  float sum[M];
#pragma unroll
  for (int i = 0; i < M; ++i) sum[i] = 0;
  // (the keys have come: else the loop would wait for them, and with them for the next rows, in every tile)
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) asm volatile("" : "+v"(k[i][s]));
  if (t_begin < t_end) write(0);
  __syncthreads();
  int buf = 0;
  for (int t0 = t_begin; t0 < t_end; t0 += stride, buf ^= 1) {
    const bool more = t0 + stride < t_end;
    if (more) read(t0 + stride);
    const int sees = old + t0 - first + 1;  // keys of the tile's first token
    v4f acc[2][M];
    auto products = [&](int q0, v4f (&out)[M]) {
#pragma unroll
      for (int i = 0; i < M; ++i) out[i] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) {
          const v4u q = *reinterpret_cast<const v4u*>(&sh.q[buf][p][place(q0 + n, 4 * s + g)]);
#pragma unroll
          for (int i = 0; i < M; ++i) out[i] = mma<TC>(q, k[i][s], out[i]);
        }
    };
    auto weights = [&](int q0, v4f (&x)[M], auto masked) {
      const v4f hi = *reinterpret_cast<const v4f*>(&sh.hi[buf][q0 + 4 * g]), f = *reinterpret_cast<const v4f*>(&sh.f[buf][q0 + 4 * g]);
      v4f c = {a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2};
      if constexpr (T == DQ_F32) c = *reinterpret_cast<const v4f*>(&sh.c[buf][q0 + 4 * g]);
      v4i token = {0, 0, 0, 0};
      if constexpr (masked()) token = *reinterpret_cast<const v4i*>(&sh.token[q0 + 4 * g]);
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = fmaf(x[i][e], c[e], -hi[e]);
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = exp2_fast(x[i][e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int limit = token[e] < t_end - t0 ? sees + token[e] : 0;
#pragma unroll
        for (int i = 0; i < M; ++i) {
          if constexpr (masked())
            sum[i] += k0 + 16 * i + n < limit ? x[i][e] * f[e] : 0.f;
          else
            sum[i] = fmaf(x[i][e], f[e], sum[i]);
        }
      }
    };
    auto tile = [&](auto masked) {
      products(0, acc[0]);
#pragma unroll
      for (int j = 0; j < QR / 16; ++j) {
        if (j + 1 < QR / 16) products(16 * j + 16, acc[(j + 1) & 1]);
        weights(16 * j, acc[j & 1], masked);
      }
    };
    if (t0 + step <= t_end && k0 + 16 * M <= sees)
      tile(std::false_type{});
    else if (k0 < sees + min(step, t_end - t0) - 1)  // (the last token sees the most)
      tile(std::true_type{});
    if (more) write(buf ^ 1);
    __syncthreads();
  }
  // Rows that are left, and those whose lse is -inf, add 0 where their products are finite, and NaN elsewhere: a wave whose sums are NaN
  // makes them once more without such rows.
  bool odd = false;
#pragma unroll
  for (int i = 0; i < M; ++i) odd |= sum[i] != sum[i];
  if (__builtin_expect(__any(odd), false)) {
#pragma unroll
    for (int i = 0; i < M; ++i) sum[i] = 0;
#pragma unroll 1
    for (int t0 = t_begin; t0 < t_end; t0 += stride) {
      const int r_end = (min(step, t_end - t0) + t0 - first) * a.group;
#pragma unroll 1
      for (int r0 = (t0 - first) * a.group; r0 < r_end; r0 += 16) add_rows<T, TC, DP>(a, m, head, first, old, r0, r_end, k0, n, g, k, sum);
    }
  }
  put_mass(a, m, b, head, part, k0, len, old, n, g, sum, bad);
}

// Adds the parts of the rows that were summed apart.
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
// A workgroup takes a sequence's kv head. The budget-th largest weight is found on whole numbers that order as the weights do:
// a histogram of kBins bins between their least and largest says in which bin it lies, another one of that bin's
// numbers where in it, until a bin is one number, or taken as a whole: three passes at most. Wave w holds (or, kHeld false, reads again for each
// pass) a run of the places, so that the list comes out ascending. Bound by latency and, for long rows, by issue: 15
// rows of 5,001 places 9 us, 256 of 16,384 21 us (3.3 and 6 of them for the reads); bit by bit, with a barrier for each, 20 and 29.

constexpr int kKeepWaves = 16;
constexpr int kBinsLog2 = 11, kBins = 1 << kBinsLog2;

// (NaN 1, below all numbers; -inf 0x7FFFFF, +inf 0xFF800000; 0 is no key's)
DQ_DEV u32 weight_key(float x) {
  const u32 b = as_u(x + 0.f);  // (-0 is 0)
  if (x != x) return 1;
  return b >> 31 ? ~b : b | 0x80000000u;
}

// The sum over the lanes before this one, and over all.
DQ_DEV int lanes_before(int x, int lane, int& all) {
  int sum = x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int y = __shfl_up(sum, m, 64);
    if (lane >= m) sum += y;
  }
  all = __builtin_amdgcn_readlane(sum, 63);
  return sum - x;
}

template <int N, bool kHeld>
__global__ __launch_bounds__(kKeepWaves * 64) void k_keep(KeepArgs a) {
  constexpr int kThreads = kKeepWaves * 64, kOwn = kBins / kThreads;
  __shared__ int bins[kBins];
  __shared__ u32 s_low[kKeepWaves], s_high[kKeepWaves];
  __shared__ int s_above[kKeepWaves], s_ties[kKeepWaves], s_found[3];
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
  auto each = [&](auto&& f) {
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < N; ++i) f(i, k[i]);
    } else {
      for (int i = 0; i < rounds; ++i) f(i, key_at(i));
    }
  };
  // the least and the largest number of those that are not kept in any case
  u32 low = ~0u, high = 0;
  each([&](int, u32 x) {
    if (x != 0) low = min(low, x);
    if (x != ~0u) high = max(high, x);
  });
  low = wave_least(low);
  high = ~wave_least(~high);
  if (lane == 0) {
    s_low[wave] = low;
    s_high[wave] = high;
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) bins[threadIdx.x * kOwn + i] = 0;
  __syncthreads();
  u32 from = ~0u, to = 0;  // the number that is looked for lies here, if any
#pragma unroll
  for (int w = 0; w < kKeepWaves; ++w) {
    from = min(from, s_low[w]);
    to = max(to, s_high[w]);
  }
  int want = budget - min(a.first + a.last, len);  // it is the want-th largest of the numbers there
  u32 least = ~0u;                                 // numbers above it or at it stay; of those at it the first, where there are ties
  bool ties = false;
  while (want > 0) {
    // (to - from + 1 numbers in bins of 2^shift)
    const int bits = 32 - __builtin_clz((to - from) | 1), shift = max(bits - kBinsLog2, 0);
    each([&](int, u32 x) {
      if (x >= from && x <= to) atomicAdd(&bins[(x - from) >> shift], 1);
    });
    __syncthreads();
    // a thread takes kOwn bins, the first thread the last ones: numbers in the bins above them
    const int at = (kThreads - 1 - (int)threadIdx.x) * kOwn;
    int own[kOwn], sum = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      sum += own[i] = bins[at + i];
      bins[at + i] = 0;
    }
    int all;
    int before = lanes_before(sum, lane, all);
    if (lane == 0) s_above[wave] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kKeepWaves; ++w)
      if (w < wave) before += s_above[w];
    if (before < want && before + sum >= want) {  // (one thread)
#pragma unroll
      for (int i = kOwn - 1; i >= 0; --i) {
        if (before < want && before + own[i] >= want) {
          s_found[0] = at + i;
          s_found[1] = before;
          s_found[2] = own[i];
        }
        before += own[i];
      }
    }
    __syncthreads();
    const int bin = s_found[0], some = s_found[2];
    want -= s_found[1];
    const u32 start = from + ((u32)bin << shift);
    if (shift == 0 || some == want) {  // (a bin of one number; or all of it stays)
      least = start;
      ties = some != want;
      break;
    }
    to = min(to, start + (1u << shift) - 1);
    from = start;
  }
  __syncthreads();
  int mine = 0, tied = 0;
  each([&](int, u32 x) { mine += __popcll(__ballot(x >= least)); });
  if (ties) each([&](int, u32 x) { tied += __popcll(__ballot(x == least)); });
  if (lane == 0) {
    s_above[wave] = mine - tied;
    s_ties[wave] = tied;
  }
  __syncthreads();
  int all_above = 0, above_before = 0, ties_before = 0;
#pragma unroll
  for (int w = 0; w < kKeepWaves; ++w) {
    all_above += s_above[w];
    if (w < wave) {
      above_before += s_above[w];
      ties_before += s_ties[w];
    }
  }
  const int room = budget - all_above;  // for ties
  int left = max(room - ties_before, 0), at = above_before + min(ties_before, room);
  const uint64_t lower = (1ull << lane) - 1;
  each([&](int i, u32 x) {
    uint64_t stays = __ballot(x >= least);
    if (ties) {
      const uint64_t tie = __ballot(x == least);
      stays = __ballot(x > least || (x == least && __popcll(tie & lower) < left));
      left -= min(left, __popcll(tie));
    }
    if (stays >> lane & 1) out[at + __popcll(stays & lower)] = (int)(base + i * 64 + lane);
    at += __popcll(stays);
  });
}

// ---- their move ------------------------------------------------------------------
// A workgroup takes the keys, or the values, of a sequence's kv head: of a list's entries up to kMoveEntries, whose addresses it first
// works out together in LDS, then their rows in runs, one run's reads under way beside the run before it. Into pages of their
// own a workgroup moves one run; in place one workgroup moves all: a run is read whole before it is written, and places
// that ascend lie at their number or behind it, so that later runs read nothing that was written. The weights, which may be
// moved in place beside keys that are not, are always one workgroup's.
//
// Into pages of their own, 1,819 of 4,017 keys, 16 sequences of 5 heads of 256 (298 MB): 61 us, 8 of them for the choice before it; 107 where the compiler
// takes 254 registers (two waves a SIMD, hence the bound of six), 143 where each lane works out its rows' addresses.

constexpr int kMoveLoads = 8;  // of 16 bytes (a weight), a thread's of a run
constexpr int kMoveEntries = 2048;

// All reads of the workgroup have come.
DQ_DEV void reads_done() {
  wait_loads();
  __syncthreads();
}

template <int kThreads>
DQ_DEV void move_weights(const int32_t* kept, int64_t count, int len, const float* mass, float* out) {
  for (int64_t i0 = 0; i0 < count; i0 += kThreads * kMoveLoads) {
    float w[kMoveLoads];
    bool moves[kMoveLoads];
#pragma unroll
    for (int u = 0; u < kMoveLoads; ++u) {
      const int64_t i = i0 + u * kThreads + threadIdx.x;
      const int place = i < count ? kept[i] : -1;
      moves[u] = place >= 0 && place < len;
      w[u] = moves[u] ? mass[place] : 0.f;
    }
    reads_done();
#pragma unroll
    for (int u = 0; u < kMoveLoads; ++u)
      if (moves[u]) out[i0 + u * kThreads + threadIdx.x] = w[u];
  }
}

template <bool kInPlace, int kThreads>
__global__ __launch_bounds__(kThreads, kInPlace ? 1 : 6) void k_compact(AttnArgs a, CompactArgs c, int lanes_log2, int runs) {
  extern __shared__ v4i s_move[];  // of an entry: page and place that it comes from (page -1: none), that it goes to
  const CacheArgs& ca = a.cache;
  const int jobs = 2 * (kInPlace ? 1 : runs) + (c.mass != nullptr);
  u32 item = blockIdx.x;
  const int h = item % ca.kv_heads;
  item /= ca.kv_heads;
  const int job = item % jobs, b = item / jobs;
  const int len = seq_len(a, b);
  const int32_t* kept = c.kept + ((int64_t)b * ca.kv_heads + h) * c.budget;
  const int most = (int)min(c.budget, (int64_t)(kInPlace ? len : a.max_len));  // (in place a list ascends: it has no more)
  if (c.mass != nullptr && job == jobs - 1) {
    const int64_t at = b * c.seq + h * c.head;
    move_weights<kThreads>(kept, most, len, c.mass + at, c.mass_out + at);
    return;
  }
  const int32_t* from = a.pages + b * a.pages_stride;
  const int32_t* to = kInPlace ? from : c.to_pages + b * c.to_stride;
  uint16_t* pool = (job & 1 ? ca.v : ca.k) + h * ca.head;
  const int rows = kThreads >> lanes_log2, r = threadIdx.x >> lanes_log2, d = 8 * (threadIdx.x & ((1 << lanes_log2) - 1));
  constexpr int kLoads = kMoveLoads;
  const int run_rows = rows * kLoads;
  auto move_of = [&](int i) {
    v4i e = {-1, 0, 0, 0};
    const int place = i < most ? kept[i] : -1;
    if (place < 0 || place >= len) return e;
    const int sp = place / ca.page_size, tp = i / ca.page_size;
    const int sid = from[sp], tid = to[tp];
    if ((u32)sid < (u32)ca.n_pages && (u32)tid < (u32)ca.n_pages) e = v4i{sid, place - sp * ca.page_size, tid, i - tp * ca.page_size};
    return e;
  };
  const bool in = d < a.dim;
  auto source = [&](v4i e) { return reinterpret_cast<const v4u*>(pool + e[0] * ca.page + e[1] * ca.token + d); };
  auto target = [&](v4i e) { return reinterpret_cast<v4u*>(pool + e[2] * ca.page + e[3] * ca.token + d); };
  if constexpr (!kInPlace) {
    const int i0 = (job >> 1) * run_rows;
    if (i0 >= most) return;
#pragma unroll 1
    for (int i = threadIdx.x; i < run_rows; i += kThreads) s_move[i] = move_of(i0 + i);
    __syncthreads();
    v4i e[kLoads];
    v4u x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) e[u] = s_move[u * rows + r];
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (in && e[u][0] >= 0) x[u] = *source(e[u]);
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (in && e[u][0] >= 0) *target(e[u]) = x[u];
  } else {
    constexpr int kEntries = kMoveEntries;
    for (int c0 = 0; c0 < most; c0 += kEntries) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kEntries / kThreads; ++u) s_move[u * kThreads + threadIdx.x] = move_of(c0 + u * kThreads + threadIdx.x);
      __syncthreads();
      const int end = min(kEntries, most - c0);
      v4u x[2][kLoads];
      auto read = [&](int i0, v4u (&y)[kLoads]) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          const v4i e = s_move[min(i0 + u * rows + r, kEntries - 1)];
          if (in && i0 + u * rows + r < end && e[0] >= 0) y[u] = *source(e);
        }
      };
      auto write = [&](int i0, v4u (&y)[kLoads]) {
        // (the run's reads have come, of all waves; those of the next one may be under way)
#pragma unroll
        for (int u = 0; u < kLoads; ++u) asm volatile("" : "+v"(y[u]) : : "memory");
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          const v4i e = s_move[min(i0 + u * rows + r, kEntries - 1)];
          if (in && i0 + u * rows + r < end && e[0] >= 0) *target(e) = y[u];
        }
      };
      read(0, x[0]);
      for (int i0 = 0; i0 < end; i0 += 2 * run_rows) {
        if (i0 + run_rows < end) read(i0 + run_rows, x[1]);
        write(i0, x[0]);
        if (i0 + run_rows >= end) break;
        if (i0 + 2 * run_rows < end) read(i0 + 2 * run_rows, x[0]);
        write(i0 + run_rows, x[1]);
      }
    }
  }
}

}  // namespace

// Rows of a sequence from which on its queries go through LDS: 8 sequences of 4,096 keys, 32 / 8 heads, us without and with: bf16 heads of
// 128, 32 / 64 / 128 / 256 rows: 16.0 and 20.1, 19.8 and 20.6, 24.7 and 21.9, 34.0 and 27.0; fp32 rows, 32 / 64 / 128: 20.7 and 21.2, 28.2 and
// 24.3, 40.1 and 29.8; heads of 64, 64 / 128 rows: 12.0 and 11.5, 15.9 and 13.3. Heads of 256 (a workgroup of
// eight waves), 64 / 128 / 256 / 512 rows: 34.7 and 36.3, 42.8 and 42.8, 57.1 and 50.2, 104 and 72; fp32 rows, 32 / 64 / 128 / 512: 45.2 and 38.9,
// 61.5 and 47.5, 94 and 60, 276 and 151; heads of 192, 256 / 512 rows: 47.6 and 48.7, 84 and 71.
template <int T>
constexpr int kManyRows = T == DQ_F32 ? 64 : 128;
template <int T>
constexpr int kManyRowsWide = T == DQ_F32 ? 64 : 256;

hipError_t launch_attention_mass(int type, int cache_type, const AttnArgs& a, const MassArgs& m, hipStream_t s) {
  const int tiles = (a.max_len + kMassKeys - 1) / kMassKeys;
  const dim3 grid((uint32_t)((int64_t)a.batch * m.splits * tiles * a.cache.kv_heads));
  const hipError_t e = by_types(type, cache_type, [&](auto tq, auto tc) {
    // (a tile holds whole tokens, whose rows are addressed from its first in 32 bits)
    constexpr int kRows = kMassRows<tq()>;
    const bool near = a.q_token < (1 << 22) && a.q_head < (1 << 22);
    // (a launch counts its threads in 32 bits, workgroups of 512 among them)
    const bool fits = a.dim <= 128 || grid.x < (1u << 23);
    const bool many = (int64_t)a.max_q * a.group >= (a.dim <= 128 ? kManyRows<tq()> : kManyRowsWide<tq()>) && a.group <= kRows && near && fits;
    const auto go = [&](auto dp) {
      if (many)
        hipLaunchKernelGGL((k_mass_many<tq(), tc(), dp()>), grid, dim3(64 * kMassWaves<dp()>), 0, s, a, m, tiles);
      else
        hipLaunchKernelGGL((k_mass<tq(), tc(), dp()>), grid, dim3(256), 0, s, a, m, tiles);
      return hipGetLastError();
    };
    if (a.dim <= 64) return go(std::integral_constant<int, 64>{});
    return a.dim <= 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 256>{});
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
  else if (k.max_len <= 8 * kLanes)
    hipLaunchKernelGGL((k_keep<8, true>), grid, block, 0, s, k);
  else if (k.max_len <= 16 * kLanes)
    hipLaunchKernelGGL((k_keep<16, true>), grid, block, 0, s, k);
  else if (k.max_len <= 64 * kLanes)
    hipLaunchKernelGGL((k_keep<64, true>), grid, block, 0, s, k);
  else
    hipLaunchKernelGGL((k_keep<1, false>), grid, block, 0, s, k);
  return hipGetLastError();
}

// Sequences and heads below which a workgroup of a move in place has 512 threads, us with 256 and with 512 (8 heads of 128, 2,048 of
// 8,192 keys, the choice before it among them): 1 / 4 / 8 / 16 / 32 sequences 39.4 and 26.9, 44.1 and 31.4, 44.7 and 36.5, 71.4 and 70.3, 119 and 126.
constexpr int64_t kFewMoves = 128;

hipError_t launch_kv_compact(const AttnArgs& a, const CompactArgs& c, hipStream_t s) {
  int log2 = 0;
  while ((8 << log2) < a.dim) ++log2;
  const int64_t rows = (256 >> log2) * kMoveLoads;
  const int runs = (int)((std::min(c.budget, (int64_t)a.max_len) + rows - 1) / rows);
  const bool in_place = c.to_pages == nullptr;
  const int64_t jobs = 2 * (in_place ? 1 : runs) + (c.mass != nullptr);
  const dim3 grid((uint32_t)(jobs * a.batch * a.cache.kv_heads));
  if (!in_place)
    hipLaunchKernelGGL((k_compact<false, 256>), grid, dim3(256), (uint32_t)rows * sizeof(v4i), s, a, c, log2, runs);
  else if (a.batch * a.cache.kv_heads < kFewMoves)
    hipLaunchKernelGGL((k_compact<true, 512>), grid, dim3(512), kMoveEntries * sizeof(v4i), s, a, c, log2, runs);
  else
    hipLaunchKernelGGL((k_compact<true, 256>), grid, dim3(256), kMoveEntries * sizeof(v4i), s, a, c, log2, runs);
  return hipGetLastError();
}

}  // namespace dq
