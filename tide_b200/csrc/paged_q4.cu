// A paged cache in 4 bits (paged_q4.cuh): new keys and values into it, with the
// heads' norms and the position rotation on the way, tokens back from it, and
// attention over it.
#include <math.h>
#include <stdio.h>

#include "attn_math.cuh"
#include "paged_q4.cuh"
#include "ragged.cuh"
#include "tc_ptx.cuh"

namespace tide {
namespace q4 {

// a / b, both positive: by 32-bit numbers, where they are (the other is a hundred
// instructions).
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 31) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// ------------------------------------------------------------------ append
// y = norm(x) turned by the angle position * inv_freq: of q, rounded to its
// type once, and of k, which is rounded to 32 bits once and goes to the cache
// with v.
//
// The codes are integers, so a key next to the border between two of them is
// one step of its group off where the last bit of a 32-bit sum is, and the
// angle of a far position has lost more than that.  A key is therefore made in
// 64 bits (the angle in turns, its whole part dropped: exact to 1e-10 at
// position 2^20).  The 64-bit pipe has time for that (7 % of it in a long prompt's
// append); a row's sines and cosines are made once for all its heads.
//
// A lane has eight neighbouring channels of a head's lower half, which are a word
// of codes, and the eight that they are turned with.  So D / 16 lanes share a head,
// and the four lanes of a group find its least and largest value in two exchanges.
//
// 32768 rows of 32 + 8 + 8 heads of 128 take 145 us (4.5 TB/s), 60 % of the issue
// slots; some 2800 warp instructions a row, half of them the codes'.  192 rows 4.1
// us, all latency.
struct AppendParams {
  const void *q, *k, *v;
  int64_t q_stride, kv_stride;
  const void *q_w, *k_w;
  float eps;
  const float *inv_freq;
  float att_scale;
  const int64_t *positions, *slot_map;
  int64_t n_map;
  const int32_t *row_ids, *n_dev;
  int64_t n_rows;
  int hq, hkv;
  void *q_out;
  unsigned char *cache;
  int64_t n_pages;
  int page;
  int32_t *err;
};

// Added to a number below 2^22, its whole part (to nearest, ties to even) is in the
// last bits.
constexpr float kRounder = 12582912.f;  // 3 * 2^22

// Two neighbouring channels in the halves of a register pair, whose sums and
// products are one instruction.
using Two = uint64_t;

template <typename T>
__device__ __forceinline__ void unpack_twos(const uint4 &v, Two (&x)[4]) {
  float f[8];
  unpack16<T>(v, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = ragged::pair(f[2 * e], f[2 * e + 1]);
}

// Least and largest value of the group of which this lane, of four neighbours, has
// eight, 0 among them; whether one of them is not finite.
__device__ __forceinline__ bool extent(const Two (&x)[4], float *lo, float *hi) {
  using namespace ragged;
  constexpr unsigned kFull = 0xffffffffu;
  float v[8];
  Two odd = 0;  // NaN where one is not finite
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    unpair(x[e], &v[2 * e], &v[2 * e + 1]);
    odd = fma2(x[e], 0, odd);
  }
  float a = min3(min3(v[0], v[1], v[2]), min3(v[3], v[4], v[5]), min3(v[6], v[7], 0.f));
  float b = max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), max3(v[6], v[7], 0.f));
  float odd0, odd1;
  unpair(odd, &odd0, &odd1);
  const unsigned who = __ballot_sync(kFull, odd0 + odd1 != 0.f);
#pragma unroll
  for (int w = 1; w < 4; w *= 2) {
    a = fminf(a, __shfl_xor_sync(kFull, a, w));
    b = fmaxf(b, __shfl_xor_sync(kFull, b, w));
  }
  *lo = a;
  *hi = b;
  return who >> (threadIdx.x & 28) & 0xfu;
}

// The group's word of codes of this lane, and its scale and zero point.
template <typename T>
__device__ __forceinline__ uint32_t quantise(const Two (&x)[4], uint32_t *par) {
  using namespace ragged;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr float kMost = kHalf ? 65504.f : 3.3895313892515355e38f;
  constexpr float kLeast = kHalf ? 0x1p-21f : 0x1p-120f;
  constexpr float kPast = kHalf ? 65520.f : 0x1.ffp127f;  // what the type rounds to infinity
  float lo, hi;
  bool odd = extent(x, &lo, &hi);
  odd |= fmaxf(hi, -lo) >= kPast;  // (a key that norm and rotation took there)
  // v / by, rounded once, with inv = 1 / by rounded once: the product may be a bit
  // off, its remainder is exact and corrects it (Markstein).  Ties are common
  // (values of eight bits over scales of four), so that bit counts.
  auto over = [](float v, float by, float inv) {
    const float q = v * inv;
    return fmaf(fmaf(-q, by, v), inv, q);
  };
  // (half of each: their difference stays within 32 bits)
  const float t = over(0.5f * hi - 0.5f * lo, 7.5f, 1.f / 7.5f);
  if (odd || t == 0.f) {
    *par = odd ? 0x7fc0u : 0u;
    return 0u;
  }
  const float s = fmaxf(__uint_as_float((__float_as_uint(t) + 0xfffffu) & 0xfff00000u), kLeast);
  const float inv = __frcp_rn(s);
  const float z = (over(-lo, s, inv) + kRounder) - kRounder;
  *par = __float_as_uint(s) >> 16 | (uint32_t)z;
  // f[e] = kRounder + code - z; below 0 a code cannot be (the least value's is z -
  // z), above 15 it can
  const Two by2 = pair(-s, -s), inv2 = pair(inv, inv), rounder2 = pair(kRounder, kRounder);
  const float most = kRounder + (15.f - z);
  float f[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const Two q = mul2(x[e], inv2);
    unpair(add2(fma2(fma2(q, by2, x[e]), inv2, q), rounder2), &f[2 * e], &f[2 * e + 1]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = fminf(f[e], most);
  if (s > kMost / 16.f) {  // next to the type's largest number: none above it
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = f[e] - kRounder;
      if (fabsf(n * s) > kMost) f[e] = n - copysignf(1.f, n) + kRounder;
    }
  }
  uint32_t word = ((uint32_t)z - 0x4b400000u) * 0x11111111u;  // (modulo 2^32)
#pragma unroll
  for (int e = 0; e < 8; ++e) word += __float_as_uint(f[e]) * (1u << (4 * (e / 2) + 16 * (e % 2)));
  return word;
}

// ROWS rows a CTA, WARPS warps a row; a warp has D / 16 lanes a head, so 4 or 8
// heads at a time, of the values, of the keys, and of the queries in turn.
template <typename T, int D, int ROWS, int WARPS>
__global__ void __launch_bounds__(32 * ROWS * WARPS, 24 / (ROWS * WARPS))
    append_kernel(const __grid_constant__ AppendParams p) {
  using namespace ragged;
  using L = Layout<D>;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr int kThreads = 32 * ROWS * WARPS;
  constexpr int kLanes = D / 16;              // of a head
  constexpr int kHeads = 32 / kLanes;         // of a warp
  constexpr int kStep = WARPS * kHeads;       // from a warp's heads to its next
  // cosine and sine of channel 8 j + e at [e][j]; of 8 j + 2 e and the next, the two
  // cosines and the two sines, in 32 bits at [e][j]
  __shared__ double2 turn[ROWS][8][kLanes];
  __shared__ float2 cosines[ROWS][4][kLanes], sines[ROWS][4][kLanes];
  __shared__ int64_t s_block[ROWS];  // the slot's block in head 0; -1: nothing to write
  __shared__ int s_token[ROWS];      // and its token there; -1: no such row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = lane % kLanes, r = warp / WARPS;
  // the first head of this lane: of the values, of the keys, which begin with the
  // warps that have the fewest values, of the queries
  const int kv_tasks = (p.hkv + kHeads - 1) / kHeads;
  const int first_v = warp % WARPS * kHeads, first_k = (warp + kv_tasks * (WARPS - 1)) % WARPS * kHeads;
  const int first_q = (warp + 2 * kv_tasks * (WARPS - 1)) % WARPS * kHeads, in = lane / kLanes;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  int64_t live = p.n_rows;
  if (p.n_dev) live = min((int64_t)max(__ldg(p.n_dev), 0), p.n_rows);
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  if (row0 >= live) return;
  const bool mine = row0 + r < live;
  const int head_blocks = p.page / kBlock;
  // this lane's channels 8 j.. and D / 2 + 8 j..
  struct Raw {
    uint4 a, b;
  };
  auto load = [&](const void *from, int64_t stride, int h, int heads) {
    Raw x{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (mine && h < heads) {
      const T *src = static_cast<const T *>(from) + (row0 + r) * stride + h * D + 8 * j;
      x.a = __ldcs(reinterpret_cast<const uint4 *>(src));
      x.b = __ldcs(reinterpret_cast<const uint4 *>(src + D / 2));
    }
    return x;
  };
  const int hq = p.q ? p.hq : 0;
  Raw next_v = load(p.v, p.kv_stride, first_v + in, p.hkv);
  Raw next_k = load(p.k, p.kv_stride, first_k + in, p.hkv);
  Raw next_q = load(p.q, p.q_stride, first_q + in, hq);
  // the rows' slots, and their angles' cosines and sines
  for (int i = threadIdx.x; i < ROWS * (D / 2); i += kThreads) {
    const int at = i / (D / 2), f = i % (D / 2);
    const int64_t row = row0 + at;
    if (row >= live) continue;
    const int64_t m = p.row_ids ? (int64_t)__ldg(p.row_ids + row) : row;
    const bool known = m >= 0 && m < p.n_map;
    if (f == 0) {
      const int64_t slot = known ? __ldg(p.slot_map + m) : -1;
      const int64_t pg = slot < 0 ? 0 : quotient(slot, p.page);
      const bool real = slot >= 0 && pg < p.n_pages;
      if (!known || (!real && slot != -1)) raise_error(p.err, TIDE_DEVERR_POSITION);
      const int tok = (int)(slot - pg * p.page);
      s_block[at] = real ? pg * p.hkv * head_blocks + tok / kBlock : -1;
      s_token[at] = !known ? -1 : real ? tok % kBlock : 0;
    }
    if (p.inv_freq && known) {
      const double turns = (double)__ldg(p.positions + m) * (double)__ldg(p.inv_freq + f) *
                           0.15915494309189533577;  // 1 / (2 pi)
      double c, s;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      c *= (double)p.att_scale;
      s *= (double)p.att_scale;
      turn[at][f % 8][f / 8] = make_double2(c, s);
      (f % 2 ? cosines[at][f % 8 / 2][f / 8].y : cosines[at][f % 8 / 2][f / 8].x) = (float)c;
      (f % 2 ? sines[at][f % 8 / 2][f / 8].y : sines[at][f % 8 / 2][f / 8].x) = (float)s;
    }
  }
  __syncthreads();
  if (!mine || s_token[r] < 0) return;
  const int tok = s_token[r];
  // where the row's token has its codes and scales in head 0
  unsigned char *const to = p.cache + s_block[r] * L::kBytes;
  const bool place = s_block[r] >= 0;
  auto store = [&](int side, int h, const Two (&x)[2][4]) {
    uint32_t par[2];
    const uint32_t word[2] = {quantise<T>(x[0], &par[0]), quantise<T>(x[1], &par[1])};
    if (!place || h >= p.hkv) return;
    unsigned char *block = to + (int64_t)h * head_blocks * L::kBytes;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      *reinterpret_cast<uint32_t *>(block + L::codes(side, tok) + a * (D / 4) + j * 4) = word[a];
      if (j % 4 == 0)
        *reinterpret_cast<uint16_t *>(block + L::scale(side, a * (D / 64) + j / 4, tok)) = (uint16_t)par[a];
    }
  };
#pragma unroll 1
  for (int h = first_v; h < p.hkv; h += kStep) {
    Two x[2][4];
    unpack_twos<T>(next_v.a, x[0]);
    unpack_twos<T>(next_v.b, x[1]);
    next_v = load(p.v, p.kv_stride, h + in + kStep, p.hkv);
    store(1, h + in, x);
  }
#pragma unroll 1
  for (int h = first_k; h < p.hkv; h += kStep) {
    float f[2][8];
    unpack16<T>(next_k.a, f[0]);
    unpack16<T>(next_k.b, f[1]);
    next_k = load(p.k, p.kv_stride, h + in + kStep, p.hkv);
    double rstd = 1.0;
    const T *w = static_cast<const T *>(p.k_w) + 8 * j;
    if (p.k_w) {
      double ss = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        ss = fma((double)f[0][e], (double)f[0][e], fma((double)f[1][e], (double)f[1][e], ss));
#pragma unroll
      for (int i = 1; i < kLanes; i *= 2) ss += __shfl_xor_sync(kFull, ss, i);
      rstd = rsqrt(ss / (double)D + (double)p.eps);
    }
    if (p.k_w || p.inv_freq) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        double a = (double)f[0][e], b = (double)f[1][e];
        if (p.k_w) {
          a *= rstd * (double)Elem<T>::to_f(w[e]);
          b *= rstd * (double)Elem<T>::to_f(w[D / 2 + e]);
        }
        if (p.inv_freq) {
          const double2 cs = turn[r][e][j];
          const double y = fma(a, cs.x, -(b * cs.y));
          b = fma(b, cs.x, a * cs.y);
          a = y;
        }
        f[0][e] = (float)a;
        f[1][e] = (float)b;
      }
    }
    Two x[2][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[a][e] = pair(f[a][2 * e], f[a][2 * e + 1]);
    store(0, h + in, x);
  }
  if (first_q >= hq) return;
  Two c[4], sn[4], minus[4];  // cosines, sines, and their negatives
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 cc = p.inv_freq ? cosines[r][e][j] : make_float2(1.f, 1.f);
    const float2 ss = p.inv_freq ? sines[r][e][j] : make_float2(0.f, 0.f);
    c[e] = pair(cc.x, cc.y);
    sn[e] = pair(ss.x, ss.y);
    minus[e] = pair(-ss.x, -ss.y);
  }
  T *const out = static_cast<T *>(p.q_out) + (row0 + r) * p.hq * D + 8 * j;
#pragma unroll 1
  for (int h = first_q; h < hq; h += kStep) {
    Two x[2][4];
    unpack_twos<T>(next_q.a, x[0]);
    unpack_twos<T>(next_q.b, x[1]);
    next_q = load(p.q, p.q_stride, h + in + kStep, hq);
    if (p.q_w) {
      Two sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fma2(x[0][e], x[0][e], fma2(x[1][e], x[1][e], sum));
      float ss, more;
      unpair(sum, &ss, &more);
      ss += more;
#pragma unroll
      for (int i = 1; i < kLanes; i *= 2) ss += __shfl_xor_sync(kFull, ss, i);
      const float rstd = rsqrtf(ss / (float)D + p.eps);
      const T *w = static_cast<const T *>(p.q_w) + 8 * j;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[a][e] = mul2(x[a][e], pair(rstd * Elem<T>::to_f(w[a * (D / 2) + 2 * e]),
                                       rstd * Elem<T>::to_f(w[a * (D / 2) + 2 * e + 1])));
    }
    if (p.inv_freq) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Two a = x[0][e], b = x[1][e];
        x[0][e] = fma2(a, c[e], mul2(b, minus[e]));
        x[1][e] = fma2(b, c[e], mul2(a, sn[e]));
      }
    }
    if (h + in < hq) {
      T *at = out + (h + in) * D;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float lo, hi;
          unpair(x[a][e], &lo, &hi);
          w[e] = pack2<T>(lo, hi);
        }
        *reinterpret_cast<uint4 *>(at + a * (D / 2)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// Zeros at every row's slot: D / 16 16-byte vectors of codes, and the scales, of
// a head, a thread each.
template <int D>
__global__ void __launch_bounds__(256) zeros_kernel(const __grid_constant__ AppendParams p) {
  using L = Layout<D>;
  constexpr int kPer = D / 16;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  int64_t live = p.n_rows;
  if (p.n_dev) live = min((int64_t)max(__ldg(p.n_dev), 0), p.n_rows);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (p.hkv * kPer);
  const int h = (int)(i / kPer % p.hkv), part = (int)(i % kPer);
  if (row >= live) return;
  const int64_t m = p.row_ids ? (int64_t)__ldg(p.row_ids + row) : row;
  const bool known = m >= 0 && m < p.n_map;
  const int64_t slot = known ? __ldg(p.slot_map + m) : -1;
  if (!known || slot < -1 || slot / p.page >= p.n_pages) {
    raise_error(p.err, TIDE_DEVERR_POSITION);
    return;
  }
  if (slot < 0) return;
  const int at = (int)(slot % p.page), side = part / (kPer / 2), vec = part % (kPer / 2);
  unsigned char *block =
      p.cache + ((slot / p.page * p.hkv + h) * (p.page / kBlock) + at / kBlock) * L::kBytes;
  *reinterpret_cast<uint4 *>(block + L::codes(side, at % kBlock) + vec * 16) = make_uint4(0, 0, 0, 0);
  *reinterpret_cast<uint16_t *>(block + L::scale(side, vec, at % kBlock)) = 0;
}

// -------------------------------------------------------------------- read
// A warp per row, eight channels a lane at a time, keys and values: four bytes of
// codes in, 16 bytes out.  Four of each are loaded before the first is stored.
// Bound by HBM: 26003 tokens of 8 heads of 128 in 25.4 us, 5.4 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    read_kernel(const unsigned char *__restrict__ cache, const int64_t *__restrict__ slots,
                int64_t n_rows, int hkv, int64_t n_pages, int page, T *__restrict__ k_out,
                T *__restrict__ v_out, int32_t *err) {
  using L = Layout<D>;
  constexpr int kWords = D / 8, kFlight = 4;
  const int lane = threadIdx.x & 31;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= n_rows) return;
  const int64_t slot = __ldg(slots + row);
  if (slot == -1) return;
  const int64_t pg = slot / page;
  if (slot < 0 || pg >= n_pages) {
    if (lane == 0) raise_error(err, TIDE_DEVERR_POSITION);
    return;
  }
  const int at = (int)(slot - pg * page), tok = at % kBlock, head_blocks = page / kBlock;
  const unsigned char *first = cache + (pg * hkv * head_blocks + at / kBlock) * L::kBytes;
  const int n = hkv * kWords;
  uint4 *const out[2] = {reinterpret_cast<uint4 *>(k_out) + row * n, reinterpret_cast<uint4 *>(v_out) + row * n};
  for (int e0 = lane; e0 < n; e0 += 32 * kFlight) {
    uint32_t w[kFlight][2], s[kFlight][2];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int e = e0 + 32 * f, word = e % kWords;
      if (e >= n) break;
      const unsigned char *block = first + (int64_t)(e / kWords) * head_blocks * L::kBytes;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        w[f][side] = __ldg(reinterpret_cast<const uint32_t *>(block + L::codes(side, tok) + word * 4));
        s[f][side] = __ldg(reinterpret_cast<const uint16_t *>(block + L::scale(side, word / 4, tok)));
      }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int e = e0 + 32 * f;
      if (e >= n) break;
#pragma unroll
      for (int side = 0; side < 2; ++side)
        out[side][e] = value8<T>(w[f][side], pars<T>(s[f][side] | s[f][side] << 16));
    }
  }
}

// ------------------------------------------------- attention of many rows
// The keys and values of each sequence as 16-bit pages in its order, for the
// tiles of paged_attention: a pass of 4.5 bits in and 16 out per value (28051 tokens
// of 8 heads of 128 in 27 us, where 2048 rows over them take 800).  Made in the tile
// kernel instead, each tile of rows would make them anew.
struct OpenParams {
  RaggedBatch batch;  // of these sequences: seq_ids and n_dev of all
  int first, n;       // of the call's sequences
  const unsigned char *cache;
  const int32_t *tables;
  int64_t max_pages;
  int n_pages, page, hkv;
  void *k, *v;
  int64_t wide;  // pages of a sequence in k and v
  int32_t *out_tables, *out_live;
  int few;       // sequences of up to so many tokens are not needed
  const int32_t *needed;  // 0: none is; NULL: not known
};
constexpr int kOpenPage = 128;  // tokens of a 16-bit page

// A warp per block of 16 tokens and head: 2 D / 32 words a lane, each 16 bytes out.
template <typename T, int D>
__global__ void __launch_bounds__(256) open_kernel(const __grid_constant__ OpenParams p) {
  using L = Layout<D>;
  constexpr int kWords = D / 8, kPer = kBlock * kWords / 32;  // words of a row; of a lane and side
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  const bool none = p.needed && __ldcg(p.needed) == 0;
  const int live = none ? 0 : live_sequences(p.batch) - p.first;
  // (the join of the tiles' splits reads it where none is needed, too)
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.out_live = min(max(live, 0), p.n);
  if (none) return;
  // eight blocks and heads a CTA, in order [sequence, block, head]
  const int per = (int)p.wide * (kOpenPage / kBlock) * p.hkv;
  const int64_t item = (int64_t)blockIdx.x * 8 + warp;
  const int i = (int)(item / per), left = (int)(item - (int64_t)i * per);
  if (i >= min(live, p.n)) return;
  const int block = left / p.hkv, h = left - block * p.hkv;
  const int seq = p.first + i;
  const int req = p.batch.seq_ids ? __ldg(p.batch.seq_ids + seq) : seq;
  // (bad bounds, a bad request or length are the attention's to flag; a sequence
  // without new tokens, which few = 0 means too, has pages that may be anything)
  int row0, end;
  if (!sequence_bounds(p.batch, seq, &row0, &end) || end - row0 <= p.few) return;
  if (req < 0 || req >= p.batch.n_requests) return;
  const int tok0 = block * kBlock;
  if (tok0 % kOpenPage == 0 && h == 0 && lane == 0)
    p.out_tables[req * p.wide + tok0 / kOpenPage] = i * (int)p.wide + tok0 / kOpenPage;
  const int kv = __ldg(p.batch.kv_lens + req);
  if (kv > p.batch.max_kv || tok0 >= kv) return;
  const int pg = __ldg(p.tables + req * p.max_pages + tok0 / p.page);
  const bool real = pg >= 0 && pg < p.n_pages;
  if (!real && lane == 0) raise_error(p.batch.err, TIDE_DEVERR_POSITION);
  const unsigned char *from =
      p.cache + (((int64_t)(real ? pg : 0) * p.hkv + h) * (p.page / kBlock) + tok0 % p.page / kBlock) * L::kBytes;
  const int64_t to = (((i * p.wide + tok0 / kOpenPage) * p.hkv + h) * kOpenPage + tok0 % kOpenPage) * kWords;
  // (the tokens past the last key of its block are opened too: they are masked)
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    uint32_t w[kPer], s[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int at = e * 32 + lane, tok = at / kWords, word = at % kWords;
      w[e] = __ldg(reinterpret_cast<const uint32_t *>(from + L::codes(side, 0)) + at);
      s[e] = __ldg(reinterpret_cast<const uint16_t *>(from + L::scale(side, word / 4, tok)));
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      reinterpret_cast<uint4 *>(side ? p.v : p.k)[to + e * 32 + lane] =
          real ? value8<T>(w[e], pars<T>(s[e] | s[e] << 16)) : make_uint4(0, 0, 0, 0);
  }
}

// --------------------------------------------------- attention of few rows
// Sequences with few rows (tokens times the query heads of a KV head).  A unit is
// up to 8 NT rows of a sequence, over the blocks of its keys in one head.  All
// blocks of all units in a row are dealt out evenly to as many CTAs as run at once,
// found from the lengths by a prefix sum that each makes, so a CTA has the end of
// one unit, some whole ones, and the beginning of another (a unit counts as
// kUnitCost blocks more, before its first); units that two or more CTAs share are
// joined by a kernel of their own, in the order of the keys.  (With a
// CTA a unit, and splits of equal length, a decode step of 192 requests left the
// SMs idle for a sixth of its time, and one of three very different requests for
// half.)  Short contexts are dealt out by whole units, and need no join.
// A CTA's four warps walk over every fourth block of its part of a unit each on
// their own, with their own running maxima, sums and outputs, and meet at its end.
// The rows are the narrow side of the products:
//   S^T[16 x 8 NT] = K Q^T,   O^T[D x 8 NT] += V^T P^T    (mma.sync m16n8k16).
// A lane makes its operands in registers from the codes, so nothing is staged as
// 16 bits.  The order of the tokens of a block, and of the channels, is free in
// both products, and chosen so that a lane reads what it needs in wide pieces:
//   row g of S is token kappa(g) = g / 2 + 4 (g % 2), row g + 8 the one 8 further;
//   k-elements of lane t (of four) of S are the D / 4 channels from D / 4 t on, in
//   one scale group;
//   rows g and g + 8 of O's tiles are the D / 8 channels from D / 8 g on, their
//   k-elements of lane t the tokens t, t + 4, t + 8, t + 12, whose scales lie side
//   by side and whose pairs of codes come from two words' halves.
// Each warp has two places for three blocks each, a bulk copy a block: one that it
// works on and one under way.  The sum of the weights, as they meet the values, is
// one more row of the values' product.
//
// What bounds it is the instructions: of a block's 420 some 260 make operands from
// codes, a shift, a mask, a difference and a product for two of them.  An ALU
// instruction takes two cycles of its pipe, and a product some nine in which it does
// little else, so 190 of the one and 17 of the other are 530 cycles of the 700 that a
// block takes a scheduler.
// 32 query heads on 8 KV heads of 128, with the join: 192 requests of 512 to 1535
// keys 71 us (3.1 TB/s), three of 9000 to 40000 keys 31 us, 16 requests of 1 to 9
// tokens over up to 2100 keys 28.5 us; two short ones 5.9 us.
constexpr int kFewWarps = 4;
constexpr int kBatch = 3;        // blocks of a place
// What beginning and ending a unit costs, in blocks (with 6, 9, 12 and 16, us: those
// 16 requests, some of them short, 30.5, 29.2, 28.5, 28.3; the 192 72.0, 71.4, 71.4,
// 71.5; one of 1000 keys 11.7, 10.3, 10.5, 10.6).
constexpr int kUnitCost = 12;
// The cost of a CTA, where there is so little (8, 16 and 32: one request of 1000 keys
// 9.6, 10.5, 12.9 us, 16 of them 15.4, 15.4, 19.3).
constexpr int kLeast = 8;

template <int D, int NT>
struct Few {
  static constexpr int kPlace = kBatch * Layout<D>::kBytes;
  static constexpr int kPitch = D + 4;                     // of a row of a warp's outputs, in its ring at the end
  static constexpr int kOutputs = 8 * NT * kPitch * 4;
  static constexpr int kRing = 2 * kPlace > kOutputs ? 2 * kPlace : (kOutputs + 127) / 128 * 128;  // of a warp
  static constexpr int kSmem = kFewWarps * kRing;
  static constexpr int kCtas = NT == 1 ? 4 : 3;  // of an SM
};

// A unit that several CTAs share, as the second of them has it.
struct Shared {
  int first, last;  // CTAs; first < 0: none
  int seq_row;      // its sequence's first packed row
  int row, rows;    // its rows among the sequence's [token, head of the group]
  int kvh;
};

struct FewParams {
  RaggedBatch batch;
  const unsigned char *cache;
  const int32_t *tables;
  int64_t max_pages;
  int n_pages, page_shift;
  const void *q;
  int64_t q_stride;
  void *out;
  float *part_o;    // [CTAs, 2, 8 NT, D]: of a unit that the CTA ends, of one that it begins
  float2 *part_ml;  // [CTAs, 2, 8 NT]: maximum (scaled, base 2), sum
  Shared *shared;   // [CTAs]: the unit that it ends
  int32_t *longer;  // whether a sequence has more than `few` tokens; or NULL
  int hq, hkv, group;
  int few;             // tokens a sequence may have
  int whole;           // units are not split
  float qs;
  uint32_t magic;      // kMagic of the rows' type
  uint32_t per_group;  // 2^31 / group, rounded up
};

// Row r / group of a sequence (exact for r < 2^17).
__device__ __forceinline__ int token_of(int r, uint32_t per_group) {
  return (int)((uint64_t)(uint32_t)r * per_group >> 31);
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  return __byte_perm(a, b, sel);
}

template <typename T>
constexpr uint32_t kOnes = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;  // two of them

// A unit, or a CTA's part of it.
struct Part {
  Sequence s;
  int seq, row;  // sequence, first of its rows
  int kvh;
  int at, nb;    // where the part begins in the unit's cost; blocks of the unit
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kFewWarps, Few<D, NT>::kCtas)
    few_rows_kernel(const __grid_constant__ FewParams p) {
  using namespace ragged;
  using L = Layout<D>;
  using F = Few<D, NT>;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr int kRowsMost = 8 * NT, kSteps = D / 16;
  constexpr int kKWords = D / 32;  // words of a lane's channels in a key
  constexpr int kVWords = D / 64;  // in a value
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ uint64_t full[kFewWarps][2];
  __shared__ float s_m[kFewWarps][kRowsMost], s_l[kFewWarps][kRowsMost];
  __shared__ long long s_sum[kFewWarps];
  __shared__ Part s_part;
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kFewWarps; ++w)
      for (int i = 0; i < 2; ++i) ptx::mbar_init(&full[w][i], 1);
    ptx::fence_mbar_init();
    s_abort = 0;
  }
  ptx::grid_dependency_wait();  // up to here this overlaps the kernel before
  ptx::grid_dependents_launch();
  const int live = live_sequences(p.batch);
  // Keys that the last of the rows of a unit, from `row` on, sees; its blocks, and
  // what it counts as where the units are dealt out.
  auto keys_of = [&](const Sequence &s, int row) {
    return s.kv - s.n + 1 + token_of(min(row + kRowsMost, s.n * p.group) - 1, p.per_group);
  };
  auto blocks_of = [&](const Sequence &s, int row) { return max((keys_of(s, row) + kBlock - 1) / kBlock, 1); };
  auto cost_of = [&](const Sequence &s, int row) { return p.whole ? 1 : blocks_of(s, row) + kUnitCost; };
  auto rows_of = [&](const Sequence &s) { return s.n <= p.few ? s.n * p.group : 0; };
  auto weight = [&](const Sequence &s) {  // of all units of a sequence
    long long w = 0;
    for (int row = 0; row < rows_of(s); row += kRowsMost) w += cost_of(s, row);
    return w * p.hkv;
  };
  long long pos, end;  // this CTA's are [pos, end) of all
  int longer;          // the first `longer` CTAs have share + 1, the others share
  long long share;
  {
    const int per = (live + 32 * kFewWarps - 1) / (32 * kFewWarps);
    const int from = min((int)threadIdx.x * per, live), to = min(from + per, live);
    long long sum = 0;
    Sequence s{};
    bool above = false;
    for (int i = from; i < to; ++i) {
      s = sequence(p.batch, i);
      sum += weight(s);
      above |= s.n > p.few;
    }
    long long upto = sum;
#pragma unroll
    for (int w = 1; w < 32; w *= 2) {
      const long long x = __shfl_up_sync(kFull, upto, w);
      if (lane >= w) upto += x;
    }
    if (lane == 31) s_sum[warp] = upto;
    above = __syncthreads_or(above);
    if (p.longer && blockIdx.x == 0 && threadIdx.x == 0) *p.longer = above;
    long long total = 0;
    for (int w = 0; w < kFewWarps; ++w) {
      if (w < warp) upto += s_sum[w];
      total += s_sum[w];
    }
    const long long least = p.whole ? 1 : kLeast;
    const int ctas = (int)min((long long)gridDim.x, (total + least - 1) / least);
    if ((int)blockIdx.x >= ctas) {
      if (threadIdx.x == 0 && !p.whole) p.shared[blockIdx.x].first = -1;
      return;
    }
    share = quotient(total, ctas);
    longer = (int)(total - share * ctas);
    pos = share * blockIdx.x + min((int)blockIdx.x, longer);
    end = pos + share + ((int)blockIdx.x < longer);
    if (pos >= upto - sum && pos < upto) {
      long long rest = pos - (upto - sum);
      for (int i = from; i < to; ++i) {
        if (per > 1) s = sequence(p.batch, i);
        for (int row = 0; row < rows_of(s); row += kRowsMost) {
          const long long c = cost_of(s, row);
          if (rest >= 0 && rest < c * p.hkv) {
            const int kvh = (int)quotient(rest, c);
            s_part = {s, i, row, kvh, (int)(rest - kvh * c), blocks_of(s, row)};
          }
          rest -= c * p.hkv;
        }
      }
    }
    __syncthreads();
  }
  auto cta_of = [&](long long cost) {
    const long long at = longer * (share + 1);
    return (int)(cost < at ? quotient(cost, share + 1) : longer + quotient(cost - at, share));
  };

  unsigned char *ring = dyn + warp * F::kRing;
  const int page = 1 << p.page_shift;
  const uint64_t once = l2_evict_first_policy();
  const int kappa = (g >> 1) + 4 * (g & 1);
  const int k_at = L::codes(0, kappa) + t * (D / 8), ks_at = L::scale(0, t * (D / 4) / kGroup, g >> 1);
  const int v_at = L::codes(1, t) + g * (D / 16), vs_at = L::scale(1, g * (D / 8) / kGroup, t);
  const float slack = kSlack / p.qs;
  const uint32_t magic = p.magic;
  uint32_t turn = 0;  // places used so far: the next is the last bit, its phase the one before
  bool starts = true;
  for (;;) {
    const Part u = s_part;
    const int pos0 = u.s.kv - u.s.n;  // keys before the first token's own
    const int kv = keys_of(u.s, u.row);
    const int rows = min(kRowsMost, u.s.n * p.group - u.row);
    const int tiles = (rows + 7) / 8;  // 8-row groups that there are
    // its blocks [b0, b1) are this CTA's
    const int left = p.whole ? 1 : u.nb + kUnitCost - u.at;  // of the unit's cost
    const int b0 = p.whole ? 0 : max(u.at - kUnitCost, 0);
    const int b1 = p.whole ? u.nb : u.nb - (int)min(max(left - (end - pos), 0ll), (long long)u.nb);
    // and this warp's b0 + warp, 4 further, ...
    const int blocks = max(0, (b1 - b0 - warp + kFewWarps - 1) / kFewWarps);
    const int block0 = b0 + warp;
    if (b1 > b0 || starts) {
      uint4 raw[NT][kKWords];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g;
        const bool valid = r < rows;
        const int tok = token_of(u.row + (valid ? r : 0), p.per_group);
        const T *q = static_cast<const T *>(p.q) + (u.s.row0 + tok) * p.q_stride +
                     (int64_t)(u.kvh * p.group + u.row + (valid ? r : 0) - tok * p.group) * D + t * (D / 4);
#pragma unroll
        for (int w = 0; w < kKWords; ++w)
          raw[nt][w] = valid ? *reinterpret_cast<const uint4 *>(q + 8 * w) : make_uint4(0, 0, 0, 0);
      }
      // where 32 blocks at a time are in the cache, one per lane, the next ones read
      // ahead; -1: a page outside it
      auto places = [&](int i0) {
        const int i = i0 + lane, at = (block0 + i * kFewWarps) * kBlock;
        if (i >= blocks || at >= kv) return -1;  // (or a unit without keys)
        const int pg = __ldg(p.tables + u.s.req * p.max_pages + (at >> p.page_shift));
        if (pg < 0 || pg >= p.n_pages) {
          raise_error(p.batch.err, TIDE_DEVERR_POSITION);
          return -1;
        }
        return (pg * p.hkv + u.kvh) * (page / kBlock) + (at & (page - 1)) / kBlock;
      };
      int base = 0, now = places(0), next = places(32);
      // blocks [i, i + kBatch) to a place, a lane each
      auto request = [&](int i, uint32_t to) {
        const int n = min(kBatch, blocks - i);
        if (n <= 0) return;
        if (i - base >= 32) {
          base += 32;
          now = next;
          next = places(base + 32);
        }
        const int k = i - base + lane;
        const int place0 = __shfl_sync(kFull, now, k & 31), place1 = __shfl_sync(kFull, next, k & 31);
        const int place = k < 32 ? place0 : place1;
        uint64_t *bar = &full[warp][to];
        unsigned char *at = ring + to * F::kPlace + lane * L::kBytes;
        const bool copy = lane < n && place >= 0;
        const int copies = __popc(__ballot_sync(kFull, copy));
        if (lane < n && place < 0)  // reads as zeros
          for (int e = 0; e < L::kBytes / 16; ++e) reinterpret_cast<uint4 *>(at)[e] = make_uint4(0, 0, 0, 0);
        __syncwarp();
        if (lane == 0) ptx::mbar_expect_tx(bar, copies * L::kBytes);
        __syncwarp();
        if (copy) ptx::bulk_load(at, p.cache + (int64_t)place * L::kBytes, L::kBytes, bar, once);
      };
      request(0, turn & 1);
      request(kBatch, (turn & 1) ^ 1);
      if (starts && !p.whole && threadIdx.x == 0) {
        Shared x{-1, -1, u.s.row0, u.row, rows, u.kvh};
        const long long block = pos - u.at + kUnitCost;  // the unit's first one's place in all
        if (b0 > 0) x.first = cta_of(block), x.last = cta_of(block + u.nb - 1);
        p.shared[blockIdx.x] = x;
      }
      starts = false;

      // Q^T: columns are rows 8 nt + g; the statistics of a column are kept by the
      // lanes whose accumulators belong to it, columns 8 nt + 2 t and one further
      uint32_t qb[NT][kSteps][2];
      int sees[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int w = 0; w < kKWords; ++w) {
          const uint4 x = raw[nt][w];
          qb[nt][2 * w][0] = x.x;
          qb[nt][2 * w][1] = x.y;
          qb[nt][2 * w + 1][0] = x.z;
          qb[nt][2 * w + 1][1] = x.w;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = min(nt * 8 + t * 2 + e, rows - 1);
          sees[nt][e] = pos0 + token_of(u.row + c, p.per_group) + 1;
        }
      }
      // (a weight is 2^(score qs + up); up is lowered where a score passes `most`)
      float o[NT][kSteps][4], oc[NT][4], up[NT][2], most[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        up[nt][0] = up[nt][1] = kLift<T>;
        most[nt][0] = most[nt][1] = -INFINITY;
        oc[nt][0] = oc[nt][1] = oc[nt][2] = oc[nt][3] = 0.f;
#pragma unroll
        for (int d = 0; d < kSteps; ++d) o[nt][d][0] = o[nt][d][1] = o[nt][d][2] = o[nt][d][3] = 0.f;
      }
      const int all_see = pos0 + token_of(u.row, p.per_group) + 1;  // keys that every row sees

      // One block at b, keys from `key` on.  masked: not all rows see all of them.
      auto work = [&](const unsigned char *b, int key, auto masked) {
        constexpr bool kMasked = decltype(masked)::value;
        uint32_t kw[2][kKWords], vw[4][kVWords];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char *at = b + k_at + 8 * h * L::kRow;
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4 *>(at);
            kw[h][0] = x.x, kw[h][1] = x.y, kw[h][2] = x.z, kw[h][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(at);
            kw[h][0] = x.x, kw[h][1] = x.y;
          }
        }
        const uint2 ks = *reinterpret_cast<const uint2 *>(b + ks_at);
        float sc[NT][4];
        {
          const uint32_t both = g & 1 ? 0x3232u : 0x1010u;
          const Pars<T> p0 = pars<T>(prmt(ks.x, 0u, both), magic), p1 = pars<T>(prmt(ks.y, 0u, both), magic);
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const int at = 2 * (k & 1);
            const uint32_t w0 = kw[0][k / 2], w1 = kw[1][k / 2];
            const uint32_t a[4] = {value2_at<T>(w0, at, p0, magic), value2_at<T>(w1, at, p1, magic),
                                   value2_at<T>(w0, at + 1, p0, magic), value2_at<T>(w1, at + 1, p1, magic)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (k == 0) mma16816_first<T>(sc[nt], a, qb[nt][k][0], qb[nt][k][1]);
              else mma16816<T>(sc[nt], a, qb[nt][k][0], qb[nt][k][1]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const unsigned char *at = b + v_at + 4 * h * L::kRow;
          if constexpr (D == 128) {
            const uint2 x = *reinterpret_cast<const uint2 *>(at);
            vw[h][0] = x.x, vw[h][1] = x.y;
          } else {
            vw[h][0] = *reinterpret_cast<const uint32_t *>(at);
          }
        }
        uint2 vs = *reinterpret_cast<const uint2 *>(b + vs_at);
        if constexpr (kMasked) {
          // A weight of 0 does not silence a NaN.  Past the last key a token's scales
          // are dropped; before it, where rows differ, those that are NaN are, and
          // added to the rows that do see them.
          auto drop = [](uint2 &x, int h) { (h < 2 ? x.x : x.y) &= h & 1 ? 0x0000ffffu : 0xffff0000u; };
          auto odd = [](const uint2 &x, int h) {
            return (((h < 2 ? x.x : x.y) >> (h & 1) * 16) & 0x7f80u) == 0x7f80u;
          };
#pragma unroll
          for (int h = 0; h < 4; ++h)
            if (key + t + 4 * h >= kv) drop(vs, h);
          if (__any_sync(kFull, odd(vs, 0) || odd(vs, 1) || odd(vs, 2) || odd(vs, 3))) {
            // rare: token by token, its scale being with lane 4 g + its number % 4
#pragma unroll 1
            for (int k = 0; k < kBlock; ++k) {
              const uint32_t two = __shfl_sync(kFull, k < 8 ? vs.x : vs.y, (lane & 28) + k % 4);
              const bool is = ((two >> (k / 4 & 1) * 16) & 0x7f80u) == 0x7f80u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int d = 0; d < kSteps; ++d)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (is && key + k < sees[nt][e & 1]) o[nt][d][e] = NAN;
            }
#pragma unroll
            for (int h = 0; h < 4; ++h)
              if (odd(vs, h)) drop(vs, h);
          }
        }
        uint32_t pt[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pt[nt][0] = pt[nt][1] = 0u;
          if (NT > 1 && nt >= tiles) continue;
          bool raise = false;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (kMasked) {  // tokens kappa and 8 further
              const int lim = sees[nt][e] - key - kappa;
              if (lim <= 0) sc[nt][e] = -INFINITY;
              if (lim <= 8) sc[nt][2 + e] = -INFINITY;
            }
            raise |= fmaxf(sc[nt][e], sc[nt][2 + e]) > most[nt][e];  // (the first keys: of -infinity)
          }
          if (__any_sync(kFull, raise)) {
            float a[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(sc[nt][e], sc[nt][2 + e]);
#pragma unroll
              for (int w = 4; w < 32; w *= 2) top = fmaxf(top, __shfl_xor_sync(kFull, top, w));
              const bool raised = top > most[nt][e];
              const float to = raised ? fmaf(-top, p.qs, kLift<T>) : up[nt][e];
              // (nothing there yet: whatever the factor)
              a[e] = most[nt][e] == -INFINITY ? 0.f : ex2(to - up[nt][e]);
              up[nt][e] = to;
              if (raised) most[nt][e] = top + slack;
              oc[nt][e] *= a[e];
            }
#pragma unroll
            for (int d = 0; d < kSteps; ++d) {
              o[nt][d][0] *= a[0];
              o[nt][d][1] *= a[1];
              o[nt][d][2] *= a[0];
              o[nt][d][3] *= a[1];
            }
          }
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = ex2(fmaf(sc[nt][e], p.qs, up[nt][e & 1]));
          pt[nt][0] = transpose8x8(pack_weights<T>(x[0], x[1]));
          pt[nt][1] = transpose8x8(pack_weights<T>(x[2], x[3]));
        }
        const Pars<T> p0 = pars<T>(vs.x, magic), p1 = pars<T>(vs.y, magic);
#pragma unroll
        for (int x = 0; x < kVWords; ++x) {
          const uint32_t lo0 = prmt(vw[0][x], vw[1][x], 0x5410u), hi0 = prmt(vw[0][x], vw[1][x], 0x7632u);
          const uint32_t lo1 = prmt(vw[2][x], vw[3][x], 0x5410u), hi1 = prmt(vw[2][x], vw[3][x], 0x7632u);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a[4] = {value2_at<T>(lo0, k, p0, magic), value2_at<T>(hi0, k, p0, magic),
                                   value2_at<T>(lo1, k, p1, magic), value2_at<T>(hi1, k, p1, magic)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][4 * x + k], a, pt[nt][0], pt[nt][1]);
          }
        }
        // the weights' sum: values of 1 in the rows of channel 0
        const uint32_t ones = g == 0 ? kOnes<T> : 0u;
        const uint32_t a[4] = {ones, 0u, ones, 0u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(oc[nt], a, pt[nt][0], pt[nt][1]);
      };

      int i = 0;
      bool lost = false;  // a wait has run out
#pragma unroll 1
      while (i < blocks) {
        const uint32_t at = turn & 1;
        if (!__all_sync(kFull, ptx::mbar_wait(&full[warp][at], turn >> 1 & 1, &s_abort))) {
          raise_error(p.batch.err, TIDE_DEVERR_TIMEOUT);
          s_abort = 1;
          lost = true;
          break;
        }
        const unsigned char *b = ring + at * F::kPlace;
        int key = (block0 + i * kFewWarps) * kBlock;
        const int upto = min(i + kBatch, blocks);
#pragma unroll 1
        for (; i < upto; ++i, b += L::kBytes, key += kFewWarps * kBlock) {
          if (key + kBlock <= all_see) work(b, key, std::false_type{});
          else work(b, key, std::true_type{});
        }
        __syncwarp();  // the place has been read
        ptx::fence_proxy_async();
        request(i + kBatch, at);
        ++turn;
      }
      if (lost && lane == 0) {  // wait for the copies in flight (bounded)
        volatile int none = 0;
        for (int e = i; e < min(blocks, i + 2 * kBatch); e += kBatch, ++turn)
          ptx::mbar_wait(&full[warp][turn & 1], turn >> 1 & 1, &none);
      }
      __syncwarp();

      // the four warps' outputs meet, [warp][row][D + 4]
      float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + t * 2 + e;
          if (g == 0) {
            s_m[warp][r] = kLift<T> - up[nt][e];
            s_l[warp][r] = oc[nt][e];
          }
#pragma unroll
          for (int d = 0; d < kSteps; ++d)
            *reinterpret_cast<float2 *>(mine + r * F::kPitch + g * (D / 8) + 2 * d) =
                make_float2(o[nt][d][e], o[nt][d][2 + e]);
        }
      __syncthreads();
      constexpr int kLanes = D / 4;  // lanes of a row, four columns each
      for (int r = threadIdx.x / kLanes; r < rows; r += 32 * kFewWarps / kLanes) {
        const int d = threadIdx.x % kLanes * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w)
          if (s_l[w][r] != 0.f) top = fmaxf(top, s_m[w][r]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
          if (s_l[w][r] == 0.f) continue;
          const float a = ex2(s_m[w][r] - top);
          const float4 y = *reinterpret_cast<const float4 *>(
              reinterpret_cast<const float *>(dyn + w * F::kRing) + r * F::kPitch + d);
          sum = fmaf(a, s_l[w][r], sum);
          x.x = fmaf(a, y.x, x.x);
          x.y = fmaf(a, y.y, x.y);
          x.z = fmaf(a, y.z, x.z);
          x.w = fmaf(a, y.w, x.w);
        }
        if (b0 > 0 || b1 < u.nb) {
          const int64_t part = (2 * (int64_t)blockIdx.x + (b0 == 0)) * kRowsMost + r;
          if (d == 0) p.part_ml[part] = make_float2(top, sum);
          *reinterpret_cast<float4 *>(p.part_o + part * D + d) = x;
        } else {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const int tok = token_of(u.row + r, p.per_group);
          const int64_t at = ((int64_t)u.s.row0 + tok) * p.hq + u.kvh * p.group + (u.row + r - tok * p.group);
          *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at * D + d) =
              make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
        }
      }
    }
    pos += left;
    if (pos >= end || *(volatile int *)&s_abort) return;
    ptx::fence_proxy_async();  // (copies go where the outputs were)
    __syncthreads();
    if (warp == 0) {  // the next unit
      const int row = u.row + kRowsMost;
      if (u.kvh + 1 < p.hkv) {
        if (lane == 0) s_part.kvh = u.kvh + 1, s_part.at = 0;
      } else if (row < u.s.n * p.group) {
        if (lane == 0) s_part = {u.s, u.seq, row, 0, 0, blocks_of(u.s, row)};
      } else {  // the next sequence that has one, 32 at a time
        for (int seq = u.seq + 1; seq < live; seq += 32) {
          Sequence s{};
          if (seq + lane < live) s = sequence(p.batch, seq + lane);
          const unsigned have = __ballot_sync(kFull, rows_of(s) > 0);
          if (have) {
            if (lane == __ffs(have) - 1) s_part = {s, seq + lane, 0, 0, 0, blocks_of(s, 0)};
            break;
          }
        }
      }
    }
    __syncthreads();
  }
}

// Joins the parts of the units that CTAs share, a CTA of this kernel for the second
// of them: with M = max m_i, o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.  Warps
// share the parts of a row where there are more warps than rows; eight parts each
// at a time, whose loads are all in flight before the first is used.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256)
    join_units_kernel(const Shared *__restrict__ shared, const float *__restrict__ part_o,
                      const float2 *__restrict__ part_ml, T *out, int hq, int group, uint32_t per_group) {
  constexpr int kE = D / 32, kFlight = 8, kRows = 8 * NT;
  using Vec = typename std::conditional<kE == 4, float4, float2>::type;  // a lane's columns
  __shared__ float s_m[8], s_l[8], s_o[8][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  const Shared u = shared[blockIdx.x];
  if (u.first < 0 || u.first + 1 != (int)blockIdx.x) return;
  const int parts = u.last - u.first + 1;
  const int per = u.rows > 4 ? 1 : u.rows > 2 ? 2 : u.rows > 1 ? 4 : 8;  // warps of a row
  for (int r0 = 0; r0 < u.rows; r0 += 8 / per) {
    const int r = r0 + warp / per;
    float m = -INFINITY, l = 0.f, o[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] = 0.f;
    for (int i0 = warp % per; r < u.rows && i0 < parts; i0 += per * kFlight) {
      float2 ml[kFlight];
      __align__(16) float x[kFlight][kE];
#pragma unroll
      for (int b = 0; b < kFlight; ++b) {
        const int i = min(i0 + b * per, parts - 1);
        const int64_t at = (2 * (int64_t)(u.first + i) + (i == 0)) * kRows + r;
        ml[b] = i0 + b * per < parts ? __ldcg(part_ml + at) : make_float2(-INFINITY, 0.f);
        *reinterpret_cast<Vec *>(x[b]) = __ldcg(reinterpret_cast<const Vec *>(part_o + at * D) + lane);
      }
      float top = m;
#pragma unroll
      for (int b = 0; b < kFlight; ++b) top = ml[b].y != 0.f ? fmaxf(top, ml[b].x) : top;
      const float a = l != 0.f ? exp2f(m - top) : 0.f;
      l *= a;
#pragma unroll
      for (int e = 0; e < kE; ++e) o[e] = l != 0.f ? o[e] * a : 0.f;
#pragma unroll
      for (int b = 0; b < kFlight; ++b) {
        if (ml[b].y == 0.f) continue;
        const float f = exp2f(ml[b].x - top);
        l = fmaf(f, ml[b].y, l);
#pragma unroll
        for (int e = 0; e < kE; ++e) o[e] = fmaf(f, x[b][e], o[e]);
      }
      m = top;
    }
    if (per > 1) {
      if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
      for (int e = 0; e < kE; ++e) s_o[warp][lane * kE + e] = o[e];
      __syncthreads();
      float top = -INFINITY;
      const int w0 = warp / per * per;
      for (int w = w0; w < w0 + per; ++w)
        if (s_l[w] != 0.f) top = fmaxf(top, s_m[w]);
      l = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e) o[e] = 0.f;
      for (int w = w0; w < w0 + per; ++w) {
        if (s_l[w] == 0.f) continue;
        const float f = exp2f(s_m[w] - top);
        l = fmaf(f, s_l[w], l);
#pragma unroll
        for (int e = 0; e < kE; ++e) o[e] = fmaf(f, s_o[w][lane * kE + e], o[e]);
      }
      __syncthreads();
    }
    if (r >= u.rows || warp % per) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int tok = token_of(u.row + r, per_group);
    T *to = out + (((int64_t)u.seq_row + tok) * hq + u.kvh * group + (u.row + r - tok * group)) * D + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; e += 2)
      reinterpret_cast<uint32_t *>(to)[e / 2] = ragged::pack2<T>(o[e] * inv, o[e + 1] * inv);
  }
}

}  // namespace q4
}  // namespace tide

namespace {

int fail(int code, const char *msg) {
  tide::set_last_error(msg);
  return code;
}

int report(cudaError_t e, const char *what) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) return TIDE_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
  return fail(TIDE_ERR_CUDA, buf);
}

template <typename... K, typename... A>
int start(const char *what, void (*kern)(K...), int64_t grid, int block, size_t smem, cudaStream_t s,
          A &&...args) {
  if (grid > INT32_MAX) return fail(TIDE_ERR_INVALID, "paged_q4: too many rows and heads");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return report(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...), what);
}

bool bad_cache(int64_t n_pages, int64_t page_size, int64_t hkv) {
  return n_pages < 1 || n_pages > INT32_MAX || hkv < 1 || hkv > 65536 || page_size < 16 ||
         page_size > (1 << 20) || page_size % 16;
}

template <typename T, int D>
int append(const tide::q4::AppendParams &p, cudaStream_t s) {
  using namespace tide::q4;
  // Warps a row, us for 32 / 8 heads of 128 and for 12 of 64 (8, 2 and 1 warps):
  // 192 rows 4.1, 4.9, 7.6 and 3.7, 4.5, 6.1; 512 rows 7.1, 6.1, 9.3 and 6.3, 5.0,
  // 6.3; 4096 rows 34.6, 24.8, 28.2 and 28.3, 16.1, 16.5; 16384 rows 125, 77, 78 and
  // 114, 54, 48; 32768 rows of the former - , 151, 145.
  if (p.n_rows >= 148 * 96)
    return start("paged_append_q4", append_kernel<T, D, 4, 1>, (p.n_rows + 3) / 4, 128, 0, s, p);
  if (p.n_rows >= 148 * 2)
    return start("paged_append_q4", append_kernel<T, D, 2, 2>, (p.n_rows + 1) / 2, 128, 0, s, p);
  return start("paged_append_q4", append_kernel<T, D, 1, 8>, p.n_rows, 256, 0, s, p);
}

// How an attention call is cut up.  Sequences of up to `few` tokens go to the
// few-rows kernel, longer ones as 16-bit pages to the tiles; a call that cannot
// have the one or the other does not launch it.
struct Plan {
  int nt;           // 8-row groups of a unit of the few-rows kernel; 0: none
  int few;
  bool whole;       // its units are not split
  int64_t ctas;
  bool tiles;       // whether the tiles run (single tokens never need them): in rounds
  int64_t wide;     // of sequences, so that the 16-bit pages of a round stay within 256 MB
  int64_t seqs;     // (or are one sequence's): pages of a sequence, sequences of a round
  size_t few_bytes, side, tables, inner, bytes;  // workspace
};

Plan plan_of(bool one_token, int64_t n_tokens, int64_t n_seqs, int64_t n_requests, int64_t hq,
             int64_t hkv, int64_t d, int64_t max_kv) {
  using namespace tide::q4;
  Plan p{};
  // The lengths are on the device; the average is known.  More rows a sequence than
  // kMostRows on average go to the tiles (16 requests over 4000 to 8000 keys, us as
  // few rows and as tiles: 32 rows 87 and 232, 64 rows 157 and 276, 128 rows 296 and
  // 316; over 500 to 1000: 28 and 34, 40 and 35, 61 and 37).  Else sequences of up to
  // twice as many rows go to the few-rows kernel, or all where the call has few rows,
  // which saves the launches of the tiles that find nothing.
  // Rows of a unit: 8 for up to as many on average, else 16 (64 requests over 1000 to
  // 2000 keys, 8 and 16: 4 rows 42 and 48 us, 8 rows 43 and 49, 12 rows 70 and 54).
  // Whole units for short contexts (us, whole and split: one request of 500 keys 8.7
  // and 10.2, of 1000 13.3 and 9.6; 64 of 250 to 500 14.7 and 19.6; 256 of those 49
  // and 48, of 500 to 1000 84 and 73).
  constexpr int64_t kMostRows = 64;
  const int64_t group = hq / hkv, rows = (n_tokens * group + n_seqs - 1) / n_seqs;
  p.nt = one_token || rows <= kMostRows ? (rows <= 8 ? 1 : 2) : 0;
  if (!one_token && n_seqs == 1 && n_tokens * group > 2 * kMostRows) p.nt = 0;
  if (p.nt) {
    p.few = (int)(one_token ? 1 : n_tokens * group <= 1024 ? n_tokens : 2 * kMostRows / group);
    if (p.few < 1) p.few = 1;
    p.whole = max_kv <= 512;
    // as many CTAs as run at once, or fewer where there is not work for so many
    const int64_t slots = 148 * (p.nt == 1 ? 4 : 3);
    int64_t units = (n_seqs + n_tokens * group / (8 * p.nt)) * hkv;
    if (units > slots * kLeast) units = slots * kLeast;  // (enough for all; the product below fits)
    const int64_t blocks = (max_kv + kBlock - 1) / kBlock;
    p.ctas = p.whole ? units : (units * ((blocks < 1 ? 1 : blocks) + kUnitCost) + kLeast - 1) / kLeast;
    if (p.ctas > slots) p.ctas = slots;
    if (!p.whole)
      p.few_bytes = (size_t)(p.ctas * (2 * 8 * p.nt * (d + 2) * 4 + (int64_t)sizeof(Shared)) + 15) / 16 * 16;
  }
  p.tiles = !one_token && (!p.nt || n_tokens > p.few);
  p.bytes = p.few_bytes;
  if (!p.tiles) return p;
  p.wide = (max_kv + tide::q4::kOpenPage - 1) / tide::q4::kOpenPage;
  if (p.wide < 1) p.wide = 1;
  const int64_t page = tide::q4::kOpenPage * hkv * d * 2;
  p.seqs = (1ll << 27) / (page * p.wide);
  if (p.seqs < 1) p.seqs = 1;
  if (p.seqs > n_seqs) p.seqs = n_seqs;
  p.side = (size_t)(p.seqs * p.wide * page);
  p.tables = (size_t)((n_requests * p.wide * 4 + 16 + 15) / 16 * 16);  // and the live count
  for (const int64_t n : {p.seqs, n_seqs % p.seqs}) {  // (the last round may be a smaller one)
    const size_t inner = tide::paged_tiles_workspace_size(n_tokens, n, hq, hkv, d, max_kv);
    if (inner > p.inner) p.inner = inner;
  }
  p.bytes += 2 * p.side + p.tables + p.inner;
  return p;
}

template <typename T, int D, int NT>
int launch_few(int64_t ctas, const tide::q4::FewParams &p, cudaStream_t s) {
  using namespace tide::q4;
  auto kern = few_rows_kernel<T, D, NT>;
  constexpr int smem = Few<D, NT>::kSmem;
  static std::atomic<uint64_t> set{0};  // per device
  const cudaError_t e = tide::allow_smem(kern, smem, set);
  if (e != cudaSuccess) return report(e, "paged_attention_q4");
  if (int rc = start("paged_attention_q4", kern, ctas, 32 * kFewWarps, smem, s, p)) return rc;
  if (ctas == 1 || p.whole) return TIDE_OK;
  return start("paged_attention_q4", join_units_kernel<T, D, NT>, ctas, 256, 0, s, (const Shared *)p.shared,
               (const float *)p.part_o, (const float2 *)p.part_ml, static_cast<T *>(p.out), p.hq, p.group,
               p.per_group);
}

template <typename T, int D>
int few_rows(int nt, int64_t ctas, const tide::q4::FewParams &p, cudaStream_t s) {
  return nt == 1 ? launch_few<T, D, 1>(ctas, p, s) : launch_few<T, D, 2>(ctas, p, s);
}

template <typename T, int D>
int open(const tide::q4::OpenParams &p, cudaStream_t s) {
  using namespace tide::q4;
  return start("paged_attention_q4", open_kernel<T, D>,
               (p.n * p.wide * (kOpenPage / kBlock) * p.hkv + 7) / 8, 256, 0, s, p);
}

}  // namespace

extern "C" int tide_paged_append_q4(int dtype, const void *q, int64_t q_row_stride, const void *k_new,
                                    const void *v_new, int64_t kv_row_stride, const void *q_norm_weight,
                                    const void *k_norm_weight, float eps, const float *inv_freq,
                                    float attention_scaling, const int64_t *positions,
                                    const int64_t *slot_map, int64_t n_slot_map, const int32_t *row_ids,
                                    const int32_t *n_rows_dev, int64_t n_rows, int64_t n_q_heads,
                                    int64_t n_kv_heads, int64_t head_dim, void *q_out, void *cache,
                                    int64_t n_pages, int64_t page_size, int32_t *error_word,
                                    tide_stream_t stream) {
  if (dtype != TIDE_DTYPE_BF16 && dtype != TIDE_DTYPE_F16)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_append_q4: dtype must be bf16 or fp16");
  if (head_dim != 64 && head_dim != 128)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_append_q4: head_dim must be 64 or 128");
  if (bad_cache(n_pages, page_size, n_kv_heads))
    return fail(TIDE_ERR_INVALID, "paged_append_q4: bad cache (page_size must be a multiple of 16)");
  if (n_rows < 0 || n_rows > INT32_MAX || n_slot_map < 0 || (!row_ids && n_slot_map < n_rows) ||
      (q && (n_q_heads < 1 || n_q_heads > 65536)))
    return fail(TIDE_ERR_INVALID, "paged_append_q4: bad sizes (rows, heads, slot map)");
  if (!q_row_stride) q_row_stride = n_q_heads * head_dim;
  if (!kv_row_stride) kv_row_stride = n_kv_heads * head_dim;
  if ((q && (q_row_stride < n_q_heads * head_dim || q_row_stride % 8)) ||
      kv_row_stride < n_kv_heads * head_dim || kv_row_stride % 8)
    return fail(TIDE_ERR_INVALID,
                "paged_append_q4: row strides must cover the heads and be multiples of 8");
  if (n_rows == 0) return TIDE_OK;
  if (!slot_map || !cache || (!k_new != !v_new) || (q && (!k_new || !q_out)) || (inv_freq && !positions))
    return fail(TIDE_ERR_INVALID, "paged_append_q4: NULL pointer");
  if (((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)q_out | (uintptr_t)cache) & 15)
    return fail(TIDE_ERR_ALIGNMENT, "paged_append_q4: rows and cache must be 16-byte aligned");
  tide::q4::AppendParams p{q, k_new, v_new, q_row_stride, kv_row_stride, q_norm_weight, k_norm_weight,
                           eps, inv_freq, attention_scaling, positions, slot_map, n_slot_map, row_ids,
                           n_rows_dev, n_rows, (int)n_q_heads, (int)n_kv_heads, q_out,
                           static_cast<unsigned char *>(cache), n_pages, (int)page_size, error_word};
  cudaStream_t s = (cudaStream_t)stream;
  if (!k_new) {
    const int64_t grid = (n_rows * n_kv_heads * (head_dim / 16) + 255) / 256;
    return head_dim == 128 ? start("paged_append_q4", tide::q4::zeros_kernel<128>, grid, 256, 0, s, p)
                           : start("paged_append_q4", tide::q4::zeros_kernel<64>, grid, 256, 0, s, p);
  }
  if (dtype == TIDE_DTYPE_BF16)
    return head_dim == 128 ? append<__nv_bfloat16, 128>(p, s) : append<__nv_bfloat16, 64>(p, s);
  return head_dim == 128 ? append<__half, 128>(p, s) : append<__half, 64>(p, s);
}

extern "C" int tide_paged_read_q4(int dtype, const void *cache, int64_t n_pages, int64_t page_size,
                                  const int64_t *slots, int64_t n_rows, int64_t n_kv_heads,
                                  int64_t head_dim, void *k_out, void *v_out, int32_t *error_word,
                                  tide_stream_t stream) {
  using namespace tide::q4;
  if (dtype != TIDE_DTYPE_BF16 && dtype != TIDE_DTYPE_F16)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_read_q4: dtype must be bf16 or fp16");
  if (head_dim != 64 && head_dim != 128)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_read_q4: head_dim must be 64 or 128");
  if (bad_cache(n_pages, page_size, n_kv_heads))
    return fail(TIDE_ERR_INVALID, "paged_read_q4: bad cache (page_size must be a multiple of 16)");
  if (n_rows < 0 || n_rows > INT32_MAX) return fail(TIDE_ERR_INVALID, "paged_read_q4: bad number of rows");
  if (n_rows == 0) return TIDE_OK;
  if (!cache || !slots || !k_out || !v_out) return fail(TIDE_ERR_INVALID, "paged_read_q4: NULL pointer");
  if (((uintptr_t)cache | (uintptr_t)k_out | (uintptr_t)v_out) & 15)
    return fail(TIDE_ERR_ALIGNMENT, "paged_read_q4: rows and cache must be 16-byte aligned");
  const int64_t grid = (n_rows + 7) / 8;
  cudaStream_t s = (cudaStream_t)stream;
  const auto *c = static_cast<const unsigned char *>(cache);
  const int hkv = (int)n_kv_heads, page = (int)page_size;
  auto run = [&](auto kern, auto *k, auto *v) {
    return start("paged_read_q4", kern, grid, 256, 0, s, c, slots, n_rows, hkv, n_pages, page, k, v, error_word);
  };
  if (dtype == TIDE_DTYPE_BF16) {
    auto *k = static_cast<__nv_bfloat16 *>(k_out), *v = static_cast<__nv_bfloat16 *>(v_out);
    return head_dim == 128 ? run(read_kernel<__nv_bfloat16, 128>, k, v)
                           : run(read_kernel<__nv_bfloat16, 64>, k, v);
  }
  auto *k = static_cast<__half *>(k_out), *v = static_cast<__half *>(v_out);
  return head_dim == 128 ? run(read_kernel<__half, 128>, k, v) : run(read_kernel<__half, 64>, k, v);
}

extern "C" size_t tide_paged_attention_q4_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t n_requests,
                                                         int64_t n_q_heads, int64_t n_kv_heads,
                                                         int64_t head_dim, int64_t max_kv_len) {
  // (the limits of the call, within which nothing below overflows)
  constexpr int64_t kMost = INT32_MAX / 2;
  if (n_tokens < 1 || n_tokens > kMost || n_seqs < 1 || n_seqs > kMost || n_requests < 0 ||
      n_requests > INT32_MAX || n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads > 65536 ||
      n_q_heads / n_kv_heads > 128 || (head_dim != 64 && head_dim != 128) || max_kv_len < 0 || max_kv_len > kMost)
    return 0;
  const size_t many = plan_of(false, n_tokens, n_seqs, n_requests, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
  if (n_tokens != n_seqs) return many;
  // (cu_seqlens or not: the larger need of the two)
  const size_t one = plan_of(true, n_tokens, n_seqs, n_requests, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
  return one > many ? one : many;
}

extern "C" int tide_paged_attention_q4(int dtype, const void *q, int64_t q_row_stride, const void *cache,
                                       int64_t n_pages, int64_t page_size, const int32_t *block_tables,
                                       int64_t max_pages, int64_t n_requests, const int32_t *kv_lens,
                                       const int32_t *cu_seqlens, const int32_t *seq_ids, int64_t n_seqs,
                                       const int32_t *n_seqs_dev, void *out, int64_t n_tokens,
                                       int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                       int64_t max_kv_len, float scale, void *workspace,
                                       size_t workspace_bytes, int32_t *error_word, tide_stream_t stream) {
  if (dtype != TIDE_DTYPE_BF16 && dtype != TIDE_DTYPE_F16)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_attention_q4: dtype must be bf16 or fp16");
  if (head_dim != 64 && head_dim != 128)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_attention_q4: head_dim must be 64 or 128");
  if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > 128 ||
      n_q_heads > 65536)
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: bad heads (1 to 128 query heads per KV head)");
  if (!(scale > 0.f) || isinf(scale))
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: scale must be positive and finite");
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2 || n_seqs < 0 || n_seqs > INT32_MAX / 2)
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: bad number of rows or sequences");
  if (!q_row_stride) q_row_stride = n_q_heads * head_dim;
  if (q_row_stride < n_q_heads * head_dim || q_row_stride % 8)
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: bad row stride (rows overlap, or not a multiple of 8)");
  if (bad_cache(n_pages, page_size, n_kv_heads) || (page_size & (page_size - 1)))
    return fail(TIDE_ERR_UNSUPPORTED, "paged_attention_q4: page_size must be a power of two of at least 16");
  if (n_pages * n_kv_heads > INT32_MAX / (page_size / 16))
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: more than 2^31 blocks of 16 tokens");
  if (max_pages < 0 || n_requests < 0 || n_requests > INT32_MAX || max_kv_len < 0 ||
      max_kv_len > INT32_MAX / 2 || (max_kv_len + page_size - 1) / page_size > max_pages)
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: bad sizes (block table, max_kv_len)");
  if ((!cu_seqlens && n_seqs != n_tokens) || (!seq_ids && n_seqs > n_requests))
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: bad number of sequences");
  if (n_tokens == 0 || n_seqs == 0) return TIDE_OK;
  if (!q || !cache || !block_tables || !kv_lens || !out)
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: NULL pointer");
  if (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)out) & 15)
    return fail(TIDE_ERR_ALIGNMENT, "paged_attention_q4: q, out and the cache must be 16-byte aligned");
  const size_t need = tide_paged_attention_q4_workspace_size(n_tokens, n_seqs, n_requests, n_q_heads,
                                                             n_kv_heads, head_dim, max_kv_len);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return fail(TIDE_ERR_WORKSPACE, "paged_attention_q4: workspace missing, too small or misaligned");
  const cudaStream_t st = (cudaStream_t)stream;
  const bool bf16 = dtype == TIDE_DTYPE_BF16, wide = head_dim == 128;
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  const Plan plan =
      plan_of(!cu_seqlens, n_tokens, n_seqs, n_requests, n_q_heads, n_kv_heads, head_dim, max_kv_len);
  if (plan.tiles && plan.wide * (tide::q4::kOpenPage / 16) * n_kv_heads > INT32_MAX)
    return fail(TIDE_ERR_INVALID, "paged_attention_q4: max_kv_len too large for so many heads");
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  const tide::RaggedBatch batch{cu_seqlens, seq_ids, kv_lens, n_seqs_dev, (int)n_seqs, (int)n_requests,
                                (int)n_tokens, (int)max_kv_len, error_word};
  int rc = TIDE_OK;
  // behind the tiles' live count: whether there is a sequence for them
  int32_t *live = plan.tiles ? reinterpret_cast<int32_t *>(ws + plan.few_bytes + 2 * plan.side) : nullptr;
  int32_t *longer = plan.tiles && plan.nt ? live + 1 : nullptr;
  if (plan.nt) {
    const int64_t group = n_q_heads / n_kv_heads, rows = plan.ctas * 2 * 8 * plan.nt;
    float *part_o = reinterpret_cast<float *>(ws);
    float2 *part_ml = reinterpret_cast<float2 *>(part_o + rows * head_dim);
    const tide::q4::FewParams f{batch, static_cast<const unsigned char *>(cache), block_tables, max_pages,
                                (int)n_pages, shift, q, q_row_stride, out, part_o, part_ml,
                                reinterpret_cast<tide::q4::Shared *>(part_ml + rows), longer, (int)n_q_heads,
                                (int)n_kv_heads, (int)group, plan.few, plan.whole,
                                scale * tide::ragged::kLog2e,
                                bf16 ? tide::q4::kMagic<__nv_bfloat16> : tide::q4::kMagic<__half>,
                                (uint32_t)(((1ll << 31) + group - 1) / group)};
    const int64_t n = plan.ctas;
    const int nt = plan.nt;
    rc = bf16 ? (wide ? few_rows<__nv_bfloat16, 128>(nt, n, f, st) : few_rows<__nv_bfloat16, 64>(nt, n, f, st))
              : (wide ? few_rows<__half, 128>(nt, n, f, st) : few_rows<__half, 64>(nt, n, f, st));
  }
  if (rc || !plan.tiles) return rc;
  ws += plan.few_bytes;
  int32_t *tables = live + 4;
  for (int64_t i = 0; i < n_seqs; i += plan.seqs) {
    const int64_t n = n_seqs - i < plan.seqs ? n_seqs - i : plan.seqs;
    const tide::q4::OpenParams o{batch, (int)i, (int)n, static_cast<const unsigned char *>(cache),
                                 block_tables, max_pages, (int)n_pages, (int)page_size, (int)n_kv_heads, ws,
                                 ws + plan.side, plan.wide, tables, live, plan.few, longer};
    rc = bf16 ? (wide ? open<__nv_bfloat16, 128>(o, st) : open<__nv_bfloat16, 64>(o, st))
              : (wide ? open<__half, 128>(o, st) : open<__half, 64>(o, st));
    if (rc) return rc;
    // sequence i of this round is request i of the call where none are named
    const int64_t skip = seq_ids ? 0 : i;
    const tide::RaggedBatch part{cu_seqlens + i, seq_ids ? seq_ids + i : nullptr, kv_lens + skip,
                                 n_seqs_dev ? live : nullptr, (int)n, (int)(n_requests - skip),
                                 (int)n_tokens, (int)max_kv_len, error_word};
    const tide::KeySource src{ws, ws + plan.side, 0, tables + skip * plan.wide, plan.wide,
                              (int)(plan.seqs * plan.wide), 7};
    static_assert(tide::q4::kOpenPage == 1 << 7, "");
    rc = tide::paged_tiles(dtype, head_dim, part, src, plan.few, longer, q, q_row_stride, out, n_q_heads,
                           n_kv_heads, scale, ws + 2 * plan.side + plan.tables, st);
    if (rc) return rc;
  }
  return TIDE_OK;
}
