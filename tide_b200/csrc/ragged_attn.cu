// Attention over ragged batches: causal attention within packed sequences,
// and of new tokens over a paged cache.
//
//   o[i, h] = sum_j e^(s_ij) v[j, h / G] / (z_i + sum_j e^(s_ij)),
//   s_ij = scale * q[i, h] . k[j, h / G],
// j over the keys that row i sees, z_i its zero keys.  One pass over the keys
// with a running maximum m, sum l and unnormalised output, fp32 throughout.
//
// A warp per (row, query head), its lanes over the head dimension.
#include <math.h>
#include <stdio.h>

#include "ragged.cuh"

namespace tide {
namespace ragged {

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  RaggedBatch batch;
  KeySource src;
  const void *q;
  int64_t q_stride;
  const int32_t *zero_keys;
  void *out;
  int hq, hkv;
  float qs;  // scale * log2(e)
};

template <typename T, int D>
__global__ void __launch_bounds__(256) row_attention_kernel(Params p) {
  constexpr int kE = D / 32;  // elements per lane
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const int live = live_sequences(p.batch);
  if (row == 0)  // a bad sequence is reported although no row finds it
    for (int i = threadIdx.x; i < live; i += blockDim.x) sequence(p.batch, i);
  const int i = sequence_of_row(p.batch, live, row);
  if (i < 0) return;
  const Sequence s = sequence(p.batch, i);
  if (!s.n) return;
  const int sees = s.kv - s.n + (row - s.row0) + 1;
  const int page = 1 << p.src.page_shift;
  for (int h = threadIdx.x >> 5; h < p.hq; h += 8) {
    const int kvh = h / (p.hq / p.hkv);
    float qv[kE], acc[kE];
    const T *q = static_cast<const T *>(p.q) + row * p.q_stride + (int64_t)h * D;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      qv[e] = Elem<T>::to_f(q[lane + 32 * e]) * p.qs;
      acc[e] = 0.f;
    }
    const int z = p.zero_keys ? max(__ldg(p.zero_keys + row), 0) : 0;
    float m = z ? 0.f : -INFINITY, l = (float)z;
    for (int j = 0; j < sees; ++j) {
      int64_t at;
      bool real = true;
      if (p.src.tables) {
        const int pg = __ldg(p.src.tables + s.req * p.src.max_pages + (j >> p.src.page_shift));
        real = pg >= 0 && pg < p.src.n_pages;
        if (!real) {
          if (lane == 0) raise_error(p.batch.err, TIDE_DEVERR_POSITION);
        }
        at = (((int64_t)pg * p.hkv + kvh) * page + (j & (page - 1))) * D;
      } else {
        at = (s.row0 + j) * p.src.row_stride + (int64_t)kvh * D;
      }
      const T *k = static_cast<const T *>(p.src.k) + at, *v = static_cast<const T *>(p.src.v) + at;
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (real) dot = fmaf(qv[e], Elem<T>::to_f(k[lane + 32 * e]), dot);
      dot = warp_sum(dot);
      const float m1 = fmaxf(m, dot), a = exp2f(m - m1), w = exp2f(dot - m1);
      l = l * a + w;
#pragma unroll
      for (int e = 0; e < kE; ++e)
        acc[e] = fmaf(acc[e], a, real ? w * Elem<T>::to_f(v[lane + 32 * e]) : 0.f);
      m = m1;
    }
    T *o = static_cast<T *>(p.out) + ((int64_t)row * p.hq + h) * D;
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // a NaN stays one
#pragma unroll
    for (int e = 0; e < kE; ++e) o[lane + 32 * e] = Elem<T>::from_f(acc[e] * inv);
  }
}

}  // namespace ragged
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

// The checks that both entry points share; 0 or a status with its message.
int check_heads(int dtype, int64_t hq, int64_t hkv, int64_t d, float scale, int64_t n_tokens,
                int64_t n_seqs) {
  if (dtype != TIDE_DTYPE_BF16 && dtype != TIDE_DTYPE_F16)
    return fail(TIDE_ERR_UNSUPPORTED, "ragged attention: dtype must be bf16 or fp16");
  if (d != 64 && d != 128)
    return fail(TIDE_ERR_UNSUPPORTED, "ragged attention: head_dim must be 64 or 128");
  if (hkv < 1 || hq < 1 || hq % hkv || hq / hkv > 128 || hq > 65536)
    return fail(TIDE_ERR_INVALID, "ragged attention: bad heads (1 to 128 query heads per KV head)");
  if (!(scale > 0.f) || isinf(scale))
    return fail(TIDE_ERR_INVALID, "ragged attention: scale must be positive and finite");
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2 || n_seqs < 0 || n_seqs > INT32_MAX / 2)
    return fail(TIDE_ERR_INVALID, "ragged attention: bad number of rows or sequences");
  return TIDE_OK;
}

int launch(int dtype, int64_t d, const tide::ragged::Params &p, cudaStream_t s) {
  using namespace tide::ragged;
  auto kern = dtype == TIDE_DTYPE_BF16
                  ? (d == 128 ? row_attention_kernel<__nv_bfloat16, 128>
                              : row_attention_kernel<__nv_bfloat16, 64>)
                  : (d == 128 ? row_attention_kernel<__half, 128> : row_attention_kernel<__half, 64>);
  kern<<<(unsigned)p.batch.n_tokens, 256, 0, s>>>(p);
  return report(cudaSuccess, "ragged attention");
}

}  // namespace

extern "C" int tide_packed_attention(int dtype, const void *q, const void *k, const void *v,
                                     int64_t q_row_stride, int64_t kv_row_stride,
                                     const int32_t *cu_seqlens, int64_t n_seqs,
                                     const int32_t *zero_keys, void *out, int64_t n_tokens,
                                     int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                     float scale, int32_t *error_word, tide_stream_t stream) {
  if (int rc = check_heads(dtype, n_q_heads, n_kv_heads, head_dim, scale, n_tokens, n_seqs)) return rc;
  if (!q_row_stride) q_row_stride = n_q_heads * head_dim;
  if (!kv_row_stride) kv_row_stride = n_kv_heads * head_dim;
  if (q_row_stride < n_q_heads * head_dim || kv_row_stride < n_kv_heads * head_dim ||
      q_row_stride % 8 || kv_row_stride % 8)
    return fail(TIDE_ERR_INVALID, "packed_attention: bad row stride (rows overlap, or not a multiple of 8)");
  if (n_tokens == 0 || n_seqs == 0) return TIDE_OK;
  if (!q || !k || !v || !cu_seqlens || !out)
    return fail(TIDE_ERR_INVALID, "packed_attention: NULL pointer");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15)
    return fail(TIDE_ERR_ALIGNMENT, "packed_attention: q, k, v and out must be 16-byte aligned");
  tide::ragged::Params p{};
  p.batch = {cu_seqlens, nullptr, nullptr, nullptr, (int)n_seqs, 0, (int)n_tokens, (int)n_tokens,
             error_word};
  p.src = {k, v, kv_row_stride, nullptr, 0, 0, 0};
  p.q = q;
  p.q_stride = q_row_stride;
  p.zero_keys = zero_keys;
  p.out = out;
  p.hq = (int)n_q_heads;
  p.hkv = (int)n_kv_heads;
  p.qs = scale * tide::ragged::kLog2e;
  return launch(dtype, head_dim, p, (cudaStream_t)stream);
}

extern "C" size_t tide_paged_attention_workspace_size(int64_t n_tokens, int64_t n_seqs,
                                                      int64_t n_q_heads, int64_t n_kv_heads,
                                                      int64_t head_dim, int64_t max_kv_len) {
  (void)n_tokens;
  (void)n_seqs;
  (void)n_q_heads;
  (void)n_kv_heads;
  (void)head_dim;
  (void)max_kv_len;
  return 0;
}

extern "C" int tide_paged_attention(int dtype, const void *q, int64_t q_row_stride,
                                    const void *k_cache, const void *v_cache, int64_t n_pages,
                                    int64_t page_size, const int32_t *block_tables,
                                    int64_t max_pages, int64_t n_requests, const int32_t *kv_lens,
                                    const int32_t *cu_seqlens, const int32_t *seq_ids,
                                    int64_t n_seqs, const int32_t *n_seqs_dev, void *out,
                                    int64_t n_tokens, int64_t n_q_heads, int64_t n_kv_heads,
                                    int64_t head_dim, int64_t max_kv_len, float scale,
                                    void *workspace, size_t workspace_bytes, int32_t *error_word,
                                    tide_stream_t stream) {
  if (int rc = check_heads(dtype, n_q_heads, n_kv_heads, head_dim, scale, n_tokens, n_seqs)) return rc;
  if (!q_row_stride) q_row_stride = n_q_heads * head_dim;
  if (q_row_stride < n_q_heads * head_dim || q_row_stride % 8)
    return fail(TIDE_ERR_INVALID, "paged_attention: bad row stride (rows overlap, or not a multiple of 8)");
  if (page_size < 16 || page_size > (1 << 20) || (page_size & (page_size - 1)))
    return fail(TIDE_ERR_UNSUPPORTED, "paged_attention: page_size must be a power of two of at least 16");
  if (n_pages < 1 || n_pages * n_kv_heads > INT32_MAX / page_size || max_pages < 0 ||
      n_requests < 0 || n_requests > INT32_MAX || max_kv_len < 0 || max_kv_len > INT32_MAX / 2 ||
      (max_kv_len + page_size - 1) / page_size > max_pages)
    return fail(TIDE_ERR_INVALID, "paged_attention: bad sizes (pages, block table, max_kv_len)");
  if ((!cu_seqlens && n_seqs != n_tokens) || (!seq_ids && n_seqs > n_requests))
    return fail(TIDE_ERR_INVALID, "paged_attention: bad number of sequences");
  if (n_tokens == 0 || n_seqs == 0) return TIDE_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !kv_lens || !out)
    return fail(TIDE_ERR_INVALID, "paged_attention: NULL pointer");
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15)
    return fail(TIDE_ERR_ALIGNMENT, "paged_attention: q, out and the caches must be 16-byte aligned");
  const size_t need = tide_paged_attention_workspace_size(n_tokens, n_seqs, n_q_heads, n_kv_heads,
                                                          head_dim, max_kv_len);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return fail(TIDE_ERR_WORKSPACE, "paged_attention: workspace missing, too small or misaligned");
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  tide::ragged::Params p{};
  p.batch = {cu_seqlens, seq_ids, kv_lens, n_seqs_dev, (int)n_seqs, (int)n_requests,
             (int)n_tokens, (int)max_kv_len, error_word};
  p.src = {k_cache, v_cache, 0, block_tables, max_pages, (int)n_pages, shift};
  p.q = q;
  p.q_stride = q_row_stride;
  p.out = out;
  p.hq = (int)n_q_heads;
  p.hkv = (int)n_kv_heads;
  p.qs = scale * tide::ragged::kLog2e;
  return launch(dtype, head_dim, p, (cudaStream_t)stream);
}
