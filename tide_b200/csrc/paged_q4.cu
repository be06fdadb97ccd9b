// A paged cache in 4 bits (paged_q4.cuh): new keys and values into it, with the
// heads' norms and the position rotation on the way, tokens back from it, and
// attention over it.
#include <math.h>
#include <stdio.h>

#include "paged_q4.cuh"
#include "ragged.cuh"
#include "tc_ptx.cuh"

namespace tide {
namespace q4 {

// ------------------------------------------------------------------ append
// y = norm(x) turned by the angle position * inv_freq: of q, rounded to its
// type once, and of k, which is rounded to 32 bits once and goes to the cache
// with v.
//
// The codes are integers, so a key next to the border between two of them is
// one step of its group off where the last bit of a 32-bit sum is, and the
// angle of a far position has lost more than that.  A key is therefore made in
// 64 bits (the angle in turns, its whole part dropped: exact to 1e-10 at
// position 2^20).  That is 24 operations of the 64-bit pipe for a key of a lane,
// two cycles each, and a sine and cosine per row and frequency, which the CTA
// makes once for all its heads; both run under the loads and stores.
//
// A lane has four neighbouring channels of a head's lower half and the four
// that they are turned with, so D / 8 lanes share a head and the eight lanes of
// a group find its least and largest value in three exchanges.
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

// x / s rounded to the nearest whole number, ties to the even one: the quotient
// by multiplication may be off by a bit, and ties are common (values of eight
// bits over scales of four), so the remainder, which is exact, decides.
__device__ __forceinline__ float nearest(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float r = fmaf(-n, s, x), a = fabsf(r), half = 0.5f * s;
  const bool odd = ((int)n & 1) != 0;
  if (a > half || (a == half && odd)) n += copysignf(1.f, r);
  return n;
}

// The group of which this lane, of eight neighbours, has four values: its codes
// as the nibbles 0, 4, 1, 5 of the result, and its scale and zero point.
template <typename T>
__device__ __forceinline__ uint32_t quantise(const float (&x)[4], uint32_t *par) {
  constexpr unsigned kFull = 0xffffffffu;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr float kMost = kHalf ? 65504.f : 3.3895313892515355e38f;
  constexpr float kLeast = kHalf ? 0x1p-21f : 0x1p-120f;
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  const bool odd = !(isfinite(x[0]) && isfinite(x[1]) && isfinite(x[2]) && isfinite(x[3]));
  const unsigned who = __ballot_sync(kFull, odd);
#pragma unroll
  for (int w = 1; w < 8; w *= 2) {
    lo = fminf(lo, __shfl_xor_sync(kFull, lo, w));
    hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, w));
  }
  if (who >> (threadIdx.x & 24) & 0xffu) {
    *par = 0x7fc0u;
    return 0u;
  }
  lo = fminf(lo, 0.f);
  hi = fmaxf(hi, 0.f);
  // (half of each: their difference stays within 32 bits)
  const float t = __fdiv_rn(0.5f * hi - 0.5f * lo, 7.5f);
  if (t == 0.f) {
    *par = 0u;
    return 0u;
  }
  const float s = fmaxf(__uint_as_float((__float_as_uint(t) + 0xfffffu) & 0xfff00000u), kLeast);
  const float inv = __frcp_rn(s);
  const float z = nearest(-lo, s, inv);
  *par = __float_as_uint(s) >> 16 | (uint32_t)z;
  uint32_t c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float n = nearest(x[e], s, inv);
    if (fabsf(n * s) > kMost) n -= copysignf(1.f, n);  // (next to the type's largest number)
    c[e] = (uint32_t)fminf(fmaxf(n + z, 0.f), 15.f);
  }
  return c[0] | c[1] << 16 | c[2] << 4 | c[3] << 20;
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
  using L = Layout<D>;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr int kLanes = D / 8;         // of a head
  constexpr int kHeads = 32 / kLanes;   // of a warp
  constexpr int kFlight = 4;            // heads of a lane, loaded before the first is used
  __shared__ double2 turn[ROWS][D / 2];  // cosine and sine
  __shared__ float2 turn32[ROWS][D / 2];
  __shared__ int64_t s_slot[ROWS];       // -1: nothing to write
  __shared__ bool s_row[ROWS];           // whether there is such a row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = lane / kLanes, j = lane % kLanes;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  int64_t live = p.n_rows;
  if (p.n_dev) live = min((int64_t)max(__ldg(p.n_dev), 0), p.n_rows);
  const int64_t row0 = (int64_t)blockIdx.x * ROWS;
  if (row0 >= live) return;
  const int q_tasks = p.q ? (p.hq + kHeads - 1) / kHeads : 0, kv_tasks = (p.hkv + kHeads - 1) / kHeads;
  const int per_row = q_tasks + 2 * kv_tasks;
  const int tasks = (int)min((int64_t)ROWS, live - row0) * per_row;
  // rows' slots; the angles' cosines and sines
  for (int i = threadIdx.x; i < ROWS * (D / 2); i += 256) {
    const int r = i / (D / 2), f = i % (D / 2);
    const int64_t row = row0 + r;
    if (row >= live) continue;
    const int64_t m = p.row_ids ? (int64_t)__ldg(p.row_ids + row) : row;
    const bool known = m >= 0 && m < p.n_map;
    if (f == 0) {
      int64_t slot = known ? __ldg(p.slot_map + m) : -1;
      if (!known || slot < -1 || slot / p.page >= p.n_pages) {
        raise_error(p.err, TIDE_DEVERR_POSITION);
        slot = -1;
      }
      s_slot[r] = slot;
      s_row[r] = known;
    }
    if (p.inv_freq && known) {
      const double turns = (double)__ldg(p.positions + m) * (double)__ldg(p.inv_freq + f) *
                           0.15915494309189533577;  // 1 / (2 pi)
      double c, s;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      c *= (double)p.att_scale;
      s *= (double)p.att_scale;
      turn[r][f] = make_double2(c, s);
      turn32[r][f] = make_float2((float)c, (float)s);
    }
  }
  bool ready = false;
  for (int t0 = warp; t0 < tasks || !ready; t0 += 8 * kFlight) {
    uint2 raw[kFlight][2];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int t = t0 + 8 * i, r = t / per_row;
      int h = t % per_row;
      const T *src = nullptr;
      raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
      if (t >= tasks) continue;
      if (h < q_tasks) {
        h = h * kHeads + head;
        if (h < p.hq) src = static_cast<const T *>(p.q) + (row0 + r) * p.q_stride + (int64_t)h * D;
      } else {
        const bool value = h >= q_tasks + kv_tasks;
        h = (h - q_tasks - (value ? kv_tasks : 0)) * kHeads + head;
        if (h < p.hkv)
          src = static_cast<const T *>(value ? p.v : p.k) + (row0 + r) * p.kv_stride + (int64_t)h * D;
      }
      if (src) {
        raw[i][0] = *reinterpret_cast<const uint2 *>(src + 4 * j);
        raw[i][1] = *reinterpret_cast<const uint2 *>(src + D / 2 + 4 * j);
      }
    }
    if (!ready) {
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int t = t0 + 8 * i, r = t / per_row;
      if (t >= tasks) break;
      int h = t % per_row;
      const int kind = h < q_tasks ? 0 : h < q_tasks + kv_tasks ? 1 : 2;
      h = (kind == 0 ? h : kind == 1 ? h - q_tasks : h - q_tasks - kv_tasks) * kHeads + head;
      float x[2][4];
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[a][e] = Elem<T>::to_f(reinterpret_cast<const T *>(&raw[i][a])[e]);
      if (kind == 0) {
        if (p.q_w) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fmaf(x[0][e], x[0][e], fmaf(x[1][e], x[1][e], ss));
#pragma unroll
          for (int w = 1; w < kLanes; w *= 2) ss += __shfl_xor_sync(kFull, ss, w);
          const float rstd = rsqrtf(ss / (float)D + p.eps);
          const T *w = static_cast<const T *>(p.q_w) + 4 * j;
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[a][e] *= rstd * Elem<T>::to_f(w[a * (D / 2) + e]);
        }
        if (p.inv_freq) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 cs = turn32[r][4 * j + e];
            const float a = x[0][e], b = x[1][e];
            x[0][e] = fmaf(a, cs.x, -b * cs.y);
            x[1][e] = fmaf(b, cs.x, a * cs.y);
          }
        }
        if (h < p.hq && s_row[r]) {
          T *to = static_cast<T *>(p.q_out) + ((row0 + r) * p.hq + h) * D + 4 * j;
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            uint2 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<T *>(&o)[e] = Elem<T>::from_f(x[a][e]);
            *reinterpret_cast<uint2 *>(to + a * (D / 2)) = o;
          }
        }
        continue;
      }
      if (kind == 1 && (p.k_w || p.inv_freq)) {
        double y[2][4];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[a][e] = (double)x[a][e];
        if (p.k_w) {
          double ss = 0.0;
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fma(y[0][e], y[0][e], fma(y[1][e], y[1][e], ss));
#pragma unroll
          for (int w = 1; w < kLanes; w *= 2) ss += __shfl_xor_sync(kFull, ss, w);
          const double rstd = rsqrt(ss / (double)D + (double)p.eps);
          const T *w = static_cast<const T *>(p.k_w) + 4 * j;
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[a][e] *= rstd * (double)Elem<T>::to_f(w[a * (D / 2) + e]);
        }
        if (p.inv_freq) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double2 cs = turn[r][4 * j + e];
            const double a = y[0][e], b = y[1][e];
            y[0][e] = fma(a, cs.x, -(b * cs.y));
            y[1][e] = fma(b, cs.x, a * cs.y);
          }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[a][e] = (float)y[a][e];
      }
      uint32_t par[2];
      const uint32_t low = quantise<T>(x[0], &par[0]), high = quantise<T>(x[1], &par[1]);
      // eight channels are two lanes': the even one stores the lower half's word
      const uint32_t other = __shfl_xor_sync(kFull, j & 1 ? low : high, 1);
      const uint32_t word = j & 1 ? high << 8 | other : low | other << 8;
      const int64_t slot = s_slot[r];
      if (slot < 0 || h >= p.hkv) continue;
      const int at = (int)(slot % p.page), side = kind - 1;
      unsigned char *block =
          p.cache + ((slot / p.page * p.hkv + h) * (p.page / kBlock) + at / kBlock) * L::kBytes;
      *reinterpret_cast<uint32_t *>(block + L::codes(side, at % kBlock) + (j & 1) * (D / 4) + j / 2 * 4) = word;
      if (j % 8 == 0) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
          *reinterpret_cast<uint16_t *>(block + L::scale(side, a * (D / 64) + j / 8, at % kBlock)) =
              (uint16_t)par[a];
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
// A thread per eight channels: four bytes of codes in, 16 bytes out.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    read_kernel(const unsigned char *__restrict__ cache, const int64_t *__restrict__ slots,
                int64_t n_rows, int hkv, int64_t n_pages, int page, T *__restrict__ k_out,
                T *__restrict__ v_out, int32_t *err) {
  using L = Layout<D>;
  constexpr int kWords = D / 8;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int word = (int)(i % kWords);
  const int64_t head = i / kWords, row = head / hkv;
  if (row >= n_rows) return;
  const int64_t slot = __ldg(slots + row);
  if (slot == -1) return;
  if (slot < 0 || slot / page >= n_pages) {
    raise_error(err, TIDE_DEVERR_POSITION);
    return;
  }
  const int at = (int)(slot % page);
  const unsigned char *block =
      cache + ((slot / page * hkv + head % hkv) * (page / kBlock) + at / kBlock) * L::kBytes;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(block + L::codes(side, at % kBlock) + word * 4);
    const uint32_t s = *reinterpret_cast<const uint16_t *>(block + L::scale(side, word / 4, at % kBlock));
    T *out = side ? v_out : k_out;
    reinterpret_cast<uint4 *>(out)[i] = value8<T>(w, pars<T>(s | s << 16));
  }
}

// ------------------------------------------------- attention of many rows
// The keys and values of each sequence as 16-bit pages in its order, for the
// tiles of paged_attention: a pass of 4.5 bits in and 16 out per value, 1 / 30 of
// the time that 2048 rows over them take.
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
};
constexpr int kOpenPage = 128;  // tokens of a 16-bit page
constexpr int kOpenTokens = 64; // of a CTA

template <typename T, int D>
__global__ void __launch_bounds__(256) open_kernel(const __grid_constant__ OpenParams p) {
  using L = Layout<D>;
  constexpr int kWords = D / 8;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  const int64_t per = p.wide * (kOpenPage / kOpenTokens);
  const int i = (int)(blockIdx.x / per);
  const int tok0 = (int)(blockIdx.x % per) * kOpenTokens;
  const int live = live_sequences(p.batch) - p.first;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.out_live = min(max(live, 0), p.n);
  if (i >= live) return;
  const int seq = p.first + i;
  const int req = p.batch.seq_ids ? __ldg(p.batch.seq_ids + seq) : seq;
  // (a bad request or length is the attention's to flag)
  if (req < 0 || req >= p.batch.n_requests) return;
  if (tok0 % kOpenPage == 0 && threadIdx.x == 0)
    p.out_tables[req * p.wide + tok0 / kOpenPage] = i * (int)p.wide + tok0 / kOpenPage;
  const int kv = __ldg(p.batch.kv_lens + req);
  if (kv > p.batch.max_kv) return;
  const int tokens = min(kv - tok0, kOpenTokens);
  for (int e = threadIdx.x; e < tokens * p.hkv * kWords; e += 256) {
    const int word = e % kWords, tok = tok0 + e / kWords % tokens, h = e / (kWords * tokens);
    const int pg = __ldg(p.tables + req * p.max_pages + tok / p.page);
    const bool real = pg >= 0 && pg < p.n_pages;
    if (!real) raise_error(p.batch.err, TIDE_DEVERR_POSITION);
    const int at = tok % p.page;
    const unsigned char *block =
        p.cache + (((int64_t)(real ? pg : 0) * p.hkv + h) * (p.page / kBlock) + at / kBlock) * L::kBytes;
    const int64_t to = (((i * p.wide + tok / kOpenPage) * p.hkv + h) * kOpenPage + tok % kOpenPage) * kWords + word;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(block + L::codes(side, at % kBlock) + word * 4);
      const uint32_t s = *reinterpret_cast<const uint16_t *>(block + L::scale(side, word / 4, at % kBlock));
      reinterpret_cast<uint4 *>(side ? p.v : p.k)[to] =
          real ? value8<T>(w, pars<T>(s | s << 16)) : make_uint4(0, 0, 0, 0);
    }
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
  // Four rows a CTA share its start and its angles' pass where there are CTAs
  // enough for every SM without that; else a row, for more warps a row.
  if (p.n_rows >= 148 * 16)
    return start("paged_append_q4", append_kernel<T, D, 4>, (p.n_rows + 3) / 4, 256, 0, s, p);
  return start("paged_append_q4", append_kernel<T, D, 1>, p.n_rows, 256, 0, s, p);
}

// How a call of the many-rows path is cut up: sequences a round, so that the
// 16-bit pages of a round stay within 1 GB (or are one sequence's).
struct Rounds {
  int64_t wide;   // 16-bit pages of a sequence
  int64_t seqs;   // of a round
  size_t side;    // bytes of the keys' (or values') pages
  size_t tables, inner, bytes;
};

Rounds rounds_of(bool one_token, int64_t n_tokens, int64_t n_seqs, int64_t n_requests, int64_t hq,
                 int64_t hkv, int64_t d, int64_t max_kv) {
  Rounds r{};
  r.wide = (max_kv + tide::q4::kOpenPage - 1) / tide::q4::kOpenPage;
  if (r.wide < 1) r.wide = 1;
  const int64_t page = tide::q4::kOpenPage * hkv * d * 2;
  r.seqs = (1ll << 29) / (page * r.wide);
  if (r.seqs < 1) r.seqs = 1;
  if (r.seqs > n_seqs) r.seqs = n_seqs;
  r.side = (size_t)(r.seqs * r.wide * page);
  r.tables = (size_t)((n_requests * r.wide * 4 + 16 + 15) / 16 * 16);  // and the live count
  for (const int64_t n : {r.seqs, n_seqs % r.seqs}) {  // (the last round may be a smaller one)
    const size_t inner =
        tide_paged_attention_workspace_size(one_token ? n : n_tokens, n, hq, hkv, d, max_kv);
    if (inner > r.inner) r.inner = inner;
  }
  r.bytes = 2 * r.side + r.tables + r.inner;
  return r;
}

template <typename T, int D>
int open(const tide::q4::OpenParams &p, cudaStream_t s) {
  using namespace tide::q4;
  return start("paged_attention_q4", open_kernel<T, D>, p.n * p.wide * (kOpenPage / kOpenTokens), 256, 0, s, p);
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
  const int64_t grid = (n_rows * n_kv_heads * (head_dim / 8) + 255) / 256;
  cudaStream_t s = (cudaStream_t)stream;
  const auto *c = static_cast<const unsigned char *>(cache);
  const int hkv = (int)n_kv_heads, page = (int)page_size;
  auto run = [&](auto kern, auto *k, auto *v) {
    return start("paged_read_q4", kern, grid, 256, 0, s, c, slots, n_rows, hkv, n_pages, page, k, v, error_word);
  };
  if (dtype == TIDE_DTYPE_BF16) {
    auto *k = static_cast<__nv_bfloat16 *>(k_out), *v = static_cast<__nv_bfloat16 *>(v_out);
    return head_dim == 128 ? run(read_kernel<__nv_bfloat16, 128>, k, v) : run(read_kernel<__nv_bfloat16, 64>, k, v);
  }
  auto *k = static_cast<__half *>(k_out), *v = static_cast<__half *>(v_out);
  return head_dim == 128 ? run(read_kernel<__half, 128>, k, v) : run(read_kernel<__half, 64>, k, v);
}

extern "C" size_t tide_paged_attention_q4_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t n_requests,
                                                         int64_t n_q_heads, int64_t n_kv_heads,
                                                         int64_t head_dim, int64_t max_kv_len) {
  if (n_tokens < 1 || n_seqs < 1 || n_requests < 0 || n_kv_heads < 1 || n_q_heads < n_kv_heads ||
      max_kv_len < 0 || n_q_heads / n_kv_heads > 128)
    return 0;
  // (cu_seqlens or not: the larger need of the two)
  const size_t one = rounds_of(true, n_tokens, n_seqs, n_requests, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
  const size_t many = rounds_of(false, n_tokens, n_seqs, n_requests, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
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
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  const Rounds r = rounds_of(!cu_seqlens, n_tokens, n_seqs, n_requests, n_q_heads, n_kv_heads, head_dim, max_kv_len);
  int32_t *live = reinterpret_cast<int32_t *>(ws + 2 * r.side);
  int32_t *tables = live + 4;
  for (int64_t i = 0; i < n_seqs; i += r.seqs) {
    const int64_t n = n_seqs - i < r.seqs ? n_seqs - i : r.seqs;
    tide::q4::OpenParams p{};
    p.batch = {cu_seqlens, seq_ids, kv_lens, n_seqs_dev, (int)n_seqs, (int)n_requests, (int)n_tokens,
               (int)max_kv_len, error_word};
    p.first = (int)i;
    p.n = (int)n;
    p.cache = static_cast<const unsigned char *>(cache);
    p.tables = block_tables;
    p.max_pages = max_pages;
    p.n_pages = (int)n_pages;
    p.page = (int)page_size;
    p.hkv = (int)n_kv_heads;
    p.k = ws;
    p.v = ws + r.side;
    p.wide = r.wide;
    p.out_tables = tables;
    p.out_live = live;
    int rc = dtype == TIDE_DTYPE_BF16
                 ? (head_dim == 128 ? open<__nv_bfloat16, 128>(p, st) : open<__nv_bfloat16, 64>(p, st))
                 : (head_dim == 128 ? open<__half, 128>(p, st) : open<__half, 64>(p, st));
    if (rc) return rc;
    // sequence i of this round is request i of the call where none are named
    const int64_t skip = seq_ids ? 0 : i;
    const int64_t row = cu_seqlens ? 0 : i;
    rc = tide_paged_attention(
        dtype, static_cast<const unsigned char *>(q) + row * q_row_stride * 2, q_row_stride, p.k, p.v,
        r.seqs * r.wide, tide::q4::kOpenPage, tables + skip * r.wide, r.wide, n_requests - skip,
        kv_lens + skip, cu_seqlens ? cu_seqlens + i : nullptr, seq_ids ? seq_ids + i : nullptr, n,
        n_seqs_dev ? live : nullptr,
        static_cast<unsigned char *>(out) + row * n_q_heads * head_dim * 2, cu_seqlens ? n_tokens : n,
        n_q_heads, n_kv_heads, head_dim, max_kv_len, scale, ws + 2 * r.side + r.tables, r.inner,
        error_word, stream);
    if (rc) return rc;
  }
  return TIDE_OK;
}
