// Ragged batches: which rows and keys each packed sequence has.  Shared by
// the attention kernels over packed sequences and over a paged cache.
#pragma once

#include <atomic>

#include "common.cuh"

namespace tide {

struct RaggedBatch {
  const int32_t *cu;       // [n_seqs + 1] packed offsets; NULL: one row per sequence
  const int32_t *seq_ids;  // [n_seqs] request of each sequence; NULL: itself
  const int32_t *kv_lens;  // [n_requests]; NULL: a sequence's keys are its own rows
  const int32_t *n_dev;    // live sequence count, or NULL
  int n_seqs;
  int n_requests;
  int n_tokens;
  int max_kv;
  int32_t *err;
};

struct Sequence {
  int row0;  // first packed row
  int n;     // rows (0: nothing to do)
  int kv;    // keys that the last row sees
  int req;   // request (row of the block table)
};

__device__ __forceinline__ int live_sequences(const RaggedBatch &b) {
  if (!b.n_dev) return b.n_seqs;
  const int n = __ldg(b.n_dev);
  if (n > b.n_seqs) raise_error(b.err, TIDE_DEVERR_COUNT);
  return min(max(n, 0), b.n_seqs);
}

// Rows [*row0, *end) of sequence i; false for bounds that are out of order or
// outside the rows.
__device__ __forceinline__ bool sequence_bounds(const RaggedBatch &b, int i, int *row0, int *end) {
  *row0 = __ldg(b.cu + i);
  *end = __ldg(b.cu + i + 1);
  return *row0 >= 0 && *end >= *row0 && *end <= b.n_tokens;
}

// Sequence i of the batch; one with bad bounds, request or length is empty
// and raises TIDE_DEVERR_POSITION.
__device__ __forceinline__ Sequence sequence(const RaggedBatch &b, int i) {
  Sequence s;
  s.row0 = i;
  s.n = 1;
  if (b.cu) {
    int end;
    const bool good = sequence_bounds(b, i, &s.row0, &end);
    s.n = good ? end - s.row0 : 0;
    if (!good) {
      raise_error(b.err, TIDE_DEVERR_POSITION);
      s.row0 = 0;
    }
  }
  s.req = i;
  s.kv = s.n;
  if (s.n && b.kv_lens) {
    if (b.seq_ids) s.req = __ldg(b.seq_ids + i);
    const bool known = s.req >= 0 && s.req < b.n_requests;
    s.kv = known ? __ldg(b.kv_lens + s.req) : -1;
    if (s.kv < 0 || s.kv > b.max_kv) {
      raise_error(b.err, TIDE_DEVERR_POSITION);
      s.n = s.kv = 0;
    }
  }
  return s;
}

// The sequence that holds packed row `row`, or -1; the same for a whole warp.
// Offsets in order: the last sequence whose start is at or before the row.  Where
// that one does not hold it (a row of no sequence, or offsets out of order, among
// which such a search can miss the row's), the first of all that does.
__device__ __forceinline__ int sequence_of_row(const RaggedBatch &b, int live, int row) {
  if (!b.cu) return row < live ? row : -1;
  auto holds = [&](int i) {
    int row0, end;
    return sequence_bounds(b, i, &row0, &end) && row0 <= row && row < end;
  };
  int lo = 0, hi = live;  // cu[lo] <= row < cu[hi], if sorted
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(b.cu + mid) <= row) lo = mid;
    else hi = mid;
  }
  if (lo < live && holds(lo)) return lo;
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < live; base += 32) {
    const unsigned who = __ballot_sync(0xffffffffu, base + lane < live && holds(base + lane));
    if (who) return base + __ffs(who) - 1;
  }
  return -1;
}

// Where the keys are: rows of a packed tensor, or pages.
struct KeySource {
  const void *k, *v;
  int64_t row_stride;      // packed: elements between rows
  const int32_t *tables;   // paged: block tables [n_requests, max_pages]
  int64_t max_pages;
  int n_pages;
  int page_shift;          // log2(page_size)
};

// The kernel's dynamic shared memory limit, raised once on every device (`set`
// has a bit for each that has it; beyond 64 devices it is raised every time).
template <typename K>
inline cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t> &set) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (set.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) set.fetch_or(bit, std::memory_order_acq_rel);
  return e;
}

void set_last_error(const char *msg);

}  // namespace tide
