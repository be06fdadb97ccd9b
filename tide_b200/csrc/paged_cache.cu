// The paged cache's bookkeeping: block tables, slot maps and packed offsets
// of a step from the requests' lengths, and the write of new keys and values.
//
// page_tables_kernel.  With the tokens held c_r (0 for a request that is
// done), the new tokens n_r and the page size P,
//   have_r = ceil(c_r / P),   need_r = ceil((c_r + n_r) / P) - have_r,
//   upto_r = need_0 + ... + need_r,
// and a request gets its pages iff upto_r <= free pages: page j of its new
// ones is entry free - 1 - (upto_r - need_r + j) of the stack.  So three
// prefix sums over the requests (tokens, pages needed, pages returned) give
// every output in parallel, and the result does not depend on the order of
// threads.  The lengths are a few KB, so this is one CTA, all latency; its
// barrier lies between the last read of what the outputs may alias or
// overlap (the lengths, the free count, the tables of requests that start
// over) and the first write of those, and makes the returned pages visible to
// the threads that hand them out again.
// Up to a slot per thread it writes the slot map and the positions too; more
// tokens are work for many SMs (65536 of them on a cluster of eight took 14 us,
// bound by the issue of its eight SMs): slot_map_kernel follows, started over
// the first one's tail.  What that one cannot see from the outputs, whether a
// request found its pages, it reads from the sign of the slot of the request's
// first token, which the first kernel has written as it will be.
//
// 256 requests of a token each take 6.4 us, 64 with 65536 tokens between them
// 11 to 12.
//
// paged_append_kernel copies 2 * kv_heads * head_dim elements per row: bound
// by HBM (32768 rows of 8 heads of 128, 43 us, 6.2 TB/s), or by latency for a
// decode step's rows (256 of them 2.5 us).
#include <stdio.h>

#include "ragged.cuh"
#include "tc_ptx.cuh"

namespace tide {
namespace pages {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
static_assert(kWarps == 32, "a lane per warp in the block scan");
constexpr int kMaxRequests = 8192;
struct Params {
  const int32_t *ctx, *add, *done;
  int n_req;
  int32_t *free_pages;
  const int32_t *n_free;
  int n_pages;
  int32_t *tables;
  int64_t max_pages;
  int page;
  int32_t *n_free_out, *kv, *cu;
  int64_t *slots, *positions;
  int64_t n_slots;
  int32_t *err;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b != 0); }

template <typename V>
__device__ __forceinline__ V warp_inclusive(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Inclusive prefix sums of three values over the block's threads, on top of
// the running totals `carry` (updated to the new totals).
__device__ __forceinline__ void block_scan(long long (&v)[3], long long (&carry)[3],
                                           long long (*s_sum)[3], int tid) {
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = warp_inclusive(v[k], lane);
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < 3; ++k) s_sum[warp][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {  // the warps' sums, one per lane
    const long long own = s_sum[lane][k];
    const long long upto = warp_inclusive(own, lane);
    v[k] += carry[k] + __shfl_sync(0xffffffffu, upto - own, warp);
    carry[k] += __shfl_sync(0xffffffffu, upto, 31);
  }
  __syncthreads();
}

// The request of packed new token t < cu[n]: cu[r] <= t < cu[r + 1].
__device__ __forceinline__ int request_of(const int32_t *cu, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) page_tables_kernel(const __grid_constant__ Params p) {
  extern __shared__ int32_t dyn[];
  // per request: packed token offset, tokens held, new pages up to and with its
  // own; with `done`, where its returned pages go and how many they are
  int32_t *s_cu = dyn;                    // [n_req + 1]
  int32_t *s_ctx = s_cu + p.n_req + 1;    // [n_req]
  int32_t *s_upto = s_ctx + p.n_req;      // [n_req]; its sign: no page was to be had
  int32_t *s_push = s_upto + p.n_req;     // [n_req]
  int32_t *s_back = s_push + p.n_req;     // [n_req]
  int32_t *s_gone = s_back + p.n_req;     // the requests that return pages, in any order
  __shared__ long long s_sum[kWarps][3];
  __shared__ int s_taken, s_n_gone;
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t room = p.max_pages * p.page;
  if (tid == 0) {
    s_taken = 0;
    s_n_gone = 0;
    s_cu[0] = 0;
  }
  ptx::grid_dependency_wait();
  if (tid == 0) ptx::grid_dependents_launch();
  int n_free = __ldcg(p.n_free);  // (used when the lengths have come too)
  const bool bad_free = n_free < 0 || n_free > p.n_pages;
  n_free = min(max(n_free, 0), p.n_pages);
  __syncthreads();

  // 1. prefix sums; the pages of the requests that are done, a warp a request
  long long carry[3] = {0, 0, 0};  // tokens, pages needed, pages returned
  for (int base = 0; base < p.n_req; base += kThreads) {
    const int r = base + tid;
    const bool in = r < p.n_req;
    int held = in ? __ldcg(p.ctx + r) : 0, add = in ? __ldcg(p.add + r) : 0;
    const bool gone = in && p.done && __ldg(p.done + r) != 0;
    if (held < 0 || add < 0 || add > p.n_slots) {
      raise_error(p.err, TIDE_DEVERR_COUNT);
      held = max(held, 0);
      if (add < 0 || add > p.n_slots) add = 0;
    }
    const int back = gone ? (int)min((int64_t)ceil_div(held, p.page), p.max_pages) : 0;
    const int ctx = gone ? 0 : held;
    const bool wide = (int64_t)ctx + add > room;  // more than a row of the table holds
    const int have = ceil_div(ctx, p.page);
    const int need = wide || !add ? 0 : (int)(((int64_t)ctx + add + p.page - 1) / p.page) - have;
    long long v[3] = {add, need, back};
    block_scan(v, carry, s_sum, tid);
    if (in) {
      s_cu[r + 1] = (int32_t)min(v[0], (long long)INT32_MAX);
      s_ctx[r] = ctx;
      // checked against the free pages below, when they are known; a request
      // whose tokens do not fit in n_slots gets none either (nor do those of
      // any later one)
      const bool past = v[0] > p.n_slots;
      s_upto[r] = wide || past ? ~(int32_t)v[1] : (int32_t)v[1];
      if (back) {
        s_push[r] = (int32_t)min((long long)n_free + v[2] - back, (long long)p.n_pages);
        s_back[r] = back;
        s_gone[atomicAdd(&s_n_gone, 1)] = r;
      }
      if (wide) raise_error(p.err, TIDE_DEVERR_PAGES);
      if (past) raise_error(p.err, TIDE_DEVERR_COUNT);
    }
  }
  if (tid == 0 && bad_free) raise_error(p.err, TIDE_DEVERR_COUNT);
  __syncthreads();
  for (int i = tid >> 5; i < s_n_gone; i += kWarps) {  // a warp per request that returns pages
    const int r = s_gone[i];
    for (int j = lane; j < s_back[r]; j += 32) {
      if ((long long)s_push[r] + j < p.n_pages)
        p.free_pages[s_push[r] + j] = __ldcg(p.tables + (int64_t)r * p.max_pages + j);
      else
        raise_error(p.err, TIDE_DEVERR_PAGES);
    }
  }
  const long long avail = min((long long)n_free + carry[2], (long long)p.n_pages);
  // which requests got their pages; how many pages are taken
  int taken = 0;
  for (int r = tid; r < p.n_req; r += kThreads) {
    const int ctx = s_ctx[r], add = s_cu[r + 1] - s_cu[r], upto = s_upto[r];
    if (upto < 0 || !add) continue;
    const int need = ceil_div(ctx + add, p.page) - ceil_div(ctx, p.page);
    if (need && upto > avail) {
      s_upto[r] = ~upto;
      raise_error(p.err, TIDE_DEVERR_PAGES);
    } else if (need) {
      taken = max(taken, upto);
    }
  }
  taken = __reduce_max_sync(0xffffffffu, taken);
  if (lane == 0 && taken) atomicMax(&s_taken, taken);
  __syncthreads();  // see the header

  // 2. lengths, offsets, free count, the first slot of every request, and the
  // table entries of the new pages, a page per thread (those of the requests
  // that got theirs are the first `taken`)
  for (int r = tid; r < p.n_req; r += kThreads) {
    const int ctx = s_ctx[r], add = s_cu[r + 1] - s_cu[r], upto = s_upto[r];
    p.kv[r] = upto < 0 ? ctx : ctx + add;
    p.cu[r + 1] = s_cu[r + 1];
    if (add && p.n_slots > kThreads && s_cu[r] < p.n_slots) {
      int64_t slot = -1;
      if (upto >= 0) {
        const int pg = ctx / p.page, have = ceil_div(ctx, p.page);
        const int need = ceil_div(ctx + add, p.page) - have;
        const int page = pg < have ? __ldcg(p.tables + (int64_t)r * p.max_pages + pg)
                                   : __ldcg(p.free_pages + (avail - 1 - (upto - need)));
        slot = (int64_t)page * p.page + ctx % p.page;
      }
      p.slots[s_cu[r]] = slot;
    }
  }
  if (tid == 0) {
    p.cu[0] = 0;
    *p.n_free_out = (int32_t)(avail - s_taken);
  }
  for (int k = tid; k < s_taken; k += kThreads) {
    int lo = 0, hi = p.n_req;  // the first request with more than k pages up to it
    while (lo < hi) {
      const int mid = (lo + hi) >> 1, upto = s_upto[mid];
      if ((upto < 0 ? ~upto : upto) > k) hi = mid;
      else lo = mid + 1;
    }
    const int have = ceil_div(s_ctx[lo], p.page);
    const int need = ceil_div(s_ctx[lo] + (s_cu[lo + 1] - s_cu[lo]), p.page) - have;
    p.tables[(int64_t)lo * p.max_pages + have + (k - (s_upto[lo] - need))] =
        __ldcg(p.free_pages + (avail - 1 - k));
  }
  if (tid >= p.n_slots || p.n_slots > kThreads) return;  // (slot_map_kernel follows)
  int64_t slot = -1, pos = 0;
  if (tid < s_cu[p.n_req]) {
    const int r = request_of(s_cu, p.n_req, tid), ctx = s_ctx[r], upto = s_upto[r];
    pos = (int64_t)ctx + (tid - s_cu[r]);
    if (upto >= 0) {
      const uint32_t at = (uint32_t)pos / (uint32_t)p.page;
      const int have = ceil_div(ctx, p.page);
      const int need = ceil_div(ctx + (s_cu[r + 1] - s_cu[r]), p.page) - have;
      const int page = (int)at < have
                           ? __ldcg(p.tables + (int64_t)r * p.max_pages + at)
                           : __ldcg(p.free_pages + (avail - 1 - (upto - need) - ((int)at - have)));
      slot = (int64_t)page * p.page + (uint32_t)pos % (uint32_t)p.page;
    }
  }
  p.slots[tid] = slot;
  p.positions[tid] = pos;
}

// 3. Slots and positions where a thread per token is more than one CTA, from
// the lengths and tables that the step leaves.
__global__ void __launch_bounds__(256) slot_map_kernel(const __grid_constant__ Params p) {
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= p.n_slots) return;
  int64_t slot = -1, pos = 0;
  if (t < __ldcg(p.cu + p.n_req)) {
    const int r = request_of(p.cu, p.n_req, (int)t);
    const int start = p.cu[r], len = __ldcg(p.kv + r);
    const bool granted = __ldcg(p.slots + start) >= 0;
    pos = (int64_t)(granted ? len - (p.cu[r + 1] - start) : len) + (t - start);
    if (granted) {
      const uint32_t at = (uint32_t)pos / (uint32_t)p.page;
      slot = (int64_t)__ldcg(p.tables + (int64_t)r * p.max_pages + at) * p.page +
             (uint32_t)pos % (uint32_t)p.page;
    }
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

// A warp per row: its 2 * hkv * d / 8 16-byte vectors, keys then values.
template <int D>
__global__ void __launch_bounds__(256)
    paged_append_kernel(const uint4 *__restrict__ k_new, const uint4 *__restrict__ v_new,
                        int64_t row_vecs, const int64_t *__restrict__ slot_map, int64_t n_map,
                        const int32_t *__restrict__ row_ids, const int32_t *__restrict__ n_dev,
                        int64_t n_rows, int hkv, uint4 *__restrict__ kc, uint4 *__restrict__ vc,
                        int64_t n_pages, int page, int32_t *err) {
  constexpr int kVecs = D / 8;  // 16-byte vectors of a head
  constexpr int kFlight = 4;    // of a lane's, loaded before the first is stored
  const int lane = threadIdx.x & 31;
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  int64_t live = n_rows;
  if (n_dev) live = min((int64_t)max(__ldg(n_dev), 0), n_rows);
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); i < live;
       i += warps) {
    const int64_t m = row_ids ? (int64_t)__ldg(row_ids + i) : i;
    if (m < 0 || m >= n_map) {
      if (lane == 0) raise_error(err, TIDE_DEVERR_POSITION);
      continue;
    }
    const int64_t slot = __ldg(slot_map + m);
    if (slot == -1) continue;
    const int64_t pg = slot / page;
    if (slot < 0 || pg >= n_pages) {
      if (lane == 0) raise_error(err, TIDE_DEVERR_POSITION);
      continue;
    }
    const int64_t dst = (pg * hkv * page + slot % page) * kVecs;  // head 0
    const int64_t head = (int64_t)page * kVecs;
    const int n = hkv * kVecs;
    for (int e0 = lane; e0 < n; e0 += 32 * kFlight) {
      uint4 a[kFlight], b[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int e = e0 + 32 * f;
        a[f] = b[f] = make_uint4(0, 0, 0, 0);
        if (k_new && e < n) a[f] = k_new[i * row_vecs + e], b[f] = v_new[i * row_vecs + e];
      }
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int e = e0 + 32 * f;
        const int64_t to = dst + (e / kVecs) * head + e % kVecs;
        if (e < n) kc[to] = a[f], vc[to] = b[f];
      }
    }
  }
}

}  // namespace pages
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

}  // namespace

extern "C" int tide_page_tables(const int32_t *context_lens, const int32_t *new_lens,
                                const int32_t *done, int64_t n_requests, int32_t *free_pages,
                                const int32_t *n_free, int64_t n_pages, int32_t *block_tables,
                                int64_t max_pages, int64_t page_size, int32_t *n_free_out,
                                int32_t *kv_lens, int32_t *cu_seqlens, int64_t *slot_map,
                                int64_t *positions, int64_t n_slots, int32_t *error_word,
                                tide_stream_t stream) {
  using namespace tide::pages;
  if (n_requests < 1 || n_requests > kMaxRequests)
    return fail(TIDE_ERR_INVALID, "page_tables: n_requests must be 1..8192");
  if (n_pages < 1 || n_pages > INT32_MAX || max_pages < 1 || page_size < 1 ||
      max_pages > INT32_MAX / page_size || max_pages > INT32_MAX / n_requests || n_slots < 0 ||
      n_slots > INT32_MAX)
    return fail(TIDE_ERR_INVALID, "page_tables: bad sizes (pages, table width, slots)");
  if (!context_lens || !new_lens || !free_pages || !n_free || !block_tables || !n_free_out ||
      !kv_lens || !cu_seqlens || (n_slots && (!slot_map || !positions)))
    return fail(TIDE_ERR_INVALID, "page_tables: NULL pointer");
  Params p{context_lens, new_lens,  done,       (int)n_requests, free_pages, n_free,
           (int)n_pages, block_tables, max_pages, (int)page_size,  n_free_out, kv_lens,
           cu_seqlens,   slot_map,  positions,  n_slots,         error_word};
  const size_t smem = ((done ? 6 : 3) * (size_t)n_requests + 1) * sizeof(int32_t);
  static std::atomic<uint64_t> set{0};
  cudaError_t e = tide::allow_smem(page_tables_kernel,
                                   (int)((6 * (size_t)kMaxRequests + 1) * sizeof(int32_t)), set);
  if (e != cudaSuccess) return report(e, "page_tables");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, page_tables_kernel, p);
  if (e == cudaSuccess && n_slots > kThreads) {
    cfg.gridDim = dim3((unsigned)((n_slots + 255) / 256), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, slot_map_kernel, p);
  }
  return report(e, "page_tables");
}

extern "C" int tide_paged_append(int dtype, const void *k_new, const void *v_new,
                                 int64_t kv_row_stride, const int64_t *slot_map,
                                 int64_t n_slot_map, const int32_t *row_ids,
                                 const int32_t *n_rows_dev, int64_t n_rows, int64_t n_kv_heads,
                                 int64_t head_dim, void *k_cache, void *v_cache, int64_t n_pages,
                                 int64_t page_size, int32_t *error_word, tide_stream_t stream) {
  using namespace tide::pages;
  if (dtype != TIDE_DTYPE_BF16 && dtype != TIDE_DTYPE_F16)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_append: dtype must be bf16 or fp16");
  if (head_dim != 64 && head_dim != 128)
    return fail(TIDE_ERR_UNSUPPORTED, "paged_append: head_dim must be 64 or 128");
  const int64_t width = n_kv_heads * head_dim;
  if (kv_row_stride == 0) kv_row_stride = width;
  if (n_rows < 0 || n_kv_heads < 1 || n_kv_heads > 65536 || kv_row_stride < width ||
      kv_row_stride % 8 || n_pages < 1 || page_size < 1 || page_size > INT32_MAX ||
      n_slot_map < 0 || (!row_ids && n_slot_map < n_rows))
    return fail(TIDE_ERR_INVALID, "paged_append: bad sizes (rows, heads, stride, pages, slot map)");
  if (n_rows == 0) return TIDE_OK;
  if (!slot_map || !k_cache || !v_cache || (!k_new != !v_new))
    return fail(TIDE_ERR_INVALID, "paged_append: NULL pointer");
  if (((uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15)
    return fail(TIDE_ERR_ALIGNMENT, "paged_append: rows and caches must be 16-byte aligned");
  int64_t blocks = (n_rows + 7) / 8;
  if (blocks > 148 * 32) blocks = 148 * 32;
  cudaStream_t s = (cudaStream_t)stream;
  auto kern = head_dim == 128 ? paged_append_kernel<128> : paged_append_kernel<64>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return report(cudaLaunchKernelEx(&cfg, kern, static_cast<const uint4 *>(k_new),
                                   static_cast<const uint4 *>(v_new), kv_row_stride / 8, slot_map,
                                   n_slot_map, row_ids, n_rows_dev, n_rows, (int)n_kv_heads,
                                   static_cast<uint4 *>(k_cache), static_cast<uint4 *>(v_cache),
                                   n_pages, (int)page_size, error_word),
                "paged_append");
}
