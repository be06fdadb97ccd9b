// Attention over ragged batches: causal attention within packed sequences,
// and of chunks of new tokens over a paged cache.
//
//   o[i, h] = sum_j e^(s_ij) v[j, h / G] / (z_i + sum_j e^(s_ij)),
//   s_ij = scale * q[i, h] . k[j, h / G],
// j over the keys that row i sees, z_i its zero keys.
//
// A tile is 128 rows: floor(128 / G) consecutive tokens of a sequence times
// the G query heads of one KV head, so that a key or value loaded serves all
// heads that share it.  A unit of work is two such tiles, one behind the
// other; a CTA per SM walks over units.  Per block of 128 keys and
// tile,
//   S[128 x 128] = Q K^T      tcgen05.mma, operands in shared memory (TMA,
//                             128-byte swizzle), S in tensor memory;
//   P = 2^(S qs - m + c)      one thread per row: running maximum m and sum l,
//                             P rounded to the rows' 16-bit type (the sum l is
//                             of the unrounded ones) and written over a half of
//                             S; c = 7 for fp16, 0 for bf16 (kLift);
//   O[128 x D] += P V         tcgen05.mma with P from tensor memory and V as
//                             it lies in shared memory (its MN-major operand).
// The chain of a tile (scores, softmax, values, the next scores) is longer than
// its share of the tensor core's time; two tiles half a period apart fill in
// for one another.  One warp issues the products of both in turn, which keeps
// them apart: with a warp each they fall into step and every phase waits for
// the other tile's same phase.  The chain is cut where it can be: the value
// product starts on three quarters of P while the last quarter's exponentials
// run, and a unit's first scores are made while the one before is written out.
//
// m is only raised, and O and l rescaled, when a row's maximum has grown by
// more than 2^8 since: larger weights cost nothing (fp32 sums), and O stays
// where it is.  So a block's weights are made with m as it was, its maximum
// beside them, and made again in the rare case that m is raised.
//
// A weight is off by half a step of its 16-bit type, relatively, as long as it
// is a normal number there.  For bf16 that is any weight that 32 bits hold.
// fp16 ends at 2^-14: a row whose largest weight lies on a key of small value
// takes its output from the others, and weights of 2^-25 and below, 40000 of
// which are 1e-3 of the row, would be rounded to nothing.  So fp16 weights, and
// with them l and the zero keys' share of it, are 2^7 times as large: the
// largest 2^(8 + 7), and half a subnormal step 2^-32 of a weight at m.
//
// What bounds it: that chain.  The products take 1390 cycles of a tile's 3130
// per block (16 of 67 cycles, and the latency of two commits), the softmax the
// rest (128 exponentials a row and thread, at 16 a cycle and SM); the tensor
// cores work 65 % of the time while a unit's blocks go by, and 50 % of the whole
// prefill below (a unit costs 4000 cycles besides its blocks, and half of a
// diagonal block is masked).  A GPU at its power limit runs this at 1.6 to 1.7
// GHz, which it reaches after a few calls.  bf16, 32 query heads on 8 KV heads
// of 128, four calls in a row and 2000: 16 prompts of 2048 in 532 and 620 us
// (1030 and 887 TFLOP/s), one of 16384 in 1.72 and 1.99 ms (1280 and 1105), 2048
// tokens over 26003 paged keys in 800 and 895 us (1130 and 1010).
//
// Roles of the warps: 0-3 and 4-7 the softmax and the output of tile 0
// and 1; 8 finds the units; 9 loads; 10 issues the products; 11 cleans the
// value blocks that not every row sees: a masked weight is 0, but 0 * NaN is
// not, so rows past the last visible key are zeroed, and a value that is not
// finite at a position that only the later rows see is zeroed, noted, and
// added to the outputs of the rows that do see it.
//
// Order of units: by the number of keys they read, most first (the level of a
// unit: positions before its end, in units of its size), so that the last
// ones to start are short.  The grid has a CTA per unit; those that run take
// over the ones that have yet to start (cluster launch control), one ahead.  A
// sequence's level range and the rank within a
// level come from counting over the sequences, so no list of units is built.
// Where the sequences' keys and values exceed what L2 holds, this goes group by
// group of consecutive sequences that fit: over all sixteen prompts of a 16 x
// 2048 prefill at once (134 MB) the kernel read 1.6 GB from HBM instead of 0.5
// and took 606 us instead of 577, at its power limit.  A batch of up to 64 MB is
// one group; the groups of a larger one have 48 MB, so that the queries and
// outputs that stream past leave them there (16 x 2048 at the power limit: 637
// us with 64 MB, 621 with 48, 621 with 32, 639 with 24; 32 x 2048: 1272, 1248,
// 1244, 1266; 20 of 200 to 4000: 984, 983, 1000, 1007).
//
// Long contexts with few rows are split over the keys (paged caches only):
// the splits' unnormalised outputs, maxima and sums go to the workspace and
// join_kernel joins them, in a fixed order.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>
#include <stdio.h>

#include <atomic>
#include <type_traits>

#include "attn_math.cuh"
#include "ragged.cuh"
#include "tc_ptx.cuh"

namespace tide {
namespace ragged {

constexpr int kRows = 128;   // rows of a tile
constexpr int kKeys = 128;   // keys of a block
constexpr int kQuarter = 32; // keys of a quarter of it
constexpr int kWarps = 12;
constexpr int kReaders = 11; // warps that read the units: all but the one that finds them
constexpr int kThreads = 32 * kWarps;
constexpr int kCached = 4;   // sequences per lane that the unit search keeps in registers
template <int D>
struct Shape {
  static constexpr int kHalves = D / 64;               // 128-byte column groups
  static constexpr uint32_t kQHalf = kRows * 128;      // bytes of a column group of a Q tile
  static constexpr uint32_t kQ = kQHalf * kHalves;     // of a Q tile
  static constexpr uint32_t kHalf = kKeys * 128;       // of a column group of a K or V block
  static constexpr uint32_t kBlock = kHalf * kHalves;  // of a K or V block
  static constexpr int kStages = D == 128 ? 4 : 8;     // K and V blocks in flight
  static constexpr uint32_t kStaging = 8 * 4096;       // 32 rows x 128 bytes per softmax warp
  static constexpr uint32_t kSmem = 2 * kQ + kStages * kBlock + kStaging + 1024;  // + alignment
};

struct Params {
  RaggedBatch batch;
  KeySource src;
  const int32_t *zero_keys;
  void *out;
  float *part_o;   // [splits, n_tokens, hq, D] (splits > 1)
  float2 *part_ml; // [splits, n_tokens, hq]: maximum (scaled, base 2), sum
  int hq, hkv;
  int group;       // query heads per KV head
  int tokens;      // of a tile: kRows / group
  int splits;
  int split_blocks;  // key blocks of a split
  int few;         // sequences of up to so many tokens go to the few-rows kernel
  int64_t group_keys;  // keys whose rows, of all KV heads, are 64 MB: up to so many are
                       // one group; three quarters of them are a group of a larger batch
  int take_over;   // whether there are more CTAs than run at once
  int boxes;       // whether a warp's 32 rows are a box of the output's map
  int behind_few;  // launched over the few-rows kernel of the same call
  const int32_t *needed;  // 0: no sequence is this kernel's; NULL: not known
  float qs;        // scale * log2(e)
};

// One unit: up to 2 * tokens tokens of a sequence, one KV head, key blocks
// [b0, b1).
struct Unit {
  int valid;
  int row0;   // packed row of the first token
  int n;      // tokens
  int pos0;   // keys before the first token's own (it sees pos0 + 1)
  int kvh;
  int req;    // row of the block table
  int key0;   // packed: row of the sequence's first key
  int b0, b1;
  int split;
};

// Tokens of tile t of the unit, and the end of its key blocks (b0 if none).
__device__ __forceinline__ int tile_tokens(const Unit &u, int tokens, int t) {
  return min(max(u.n - t * tokens, 0), tokens);
}
__device__ __forceinline__ int tile_sees(const Unit &u, int tokens, int t) {
  return u.pos0 + t * tokens + tile_tokens(u, tokens, t);  // keys its last token sees
}
__device__ __forceinline__ int tile_end(const Unit &u, int tokens, int t) {
  if (tile_tokens(u, tokens, t) == 0) return u.b0;
  const int sees = max(tile_sees(u, tokens, t), 0);
  return max(u.b0, min(u.b1, (sees + kKeys - 1) / kKeys));
}

// The rows [from, to) of value block j that the cleaner goes over: those past
// the first token's own position, up to the last key that some token of the
// unit sees, rounded up to the 16 keys that a product reads.
__device__ __forceinline__ bool cleaned_rows(const Unit &u, int sees, int j, int *from, int *to) {
  *from = max(0, u.pos0 + 1 - j * kKeys);
  *to = (min(kKeys, sees - j * kKeys) + 15) / 16 * 16;
  return *from < *to;
}

constexpr int kRing = 8;  // the most stages of a Shape

struct Shared {
  uint64_t q_full[2], q_empty[2];
  uint64_t s_full[2];
  uint64_t p_full[2][2];  // [tile]: three quarters of P, the last quarter
  uint64_t o_full[2];     // after a unit's last value product
  uint64_t u_full[2], u_empty[2];
  uint64_t drain;
  uint64_t taken;   // the answer to a request for another CTA's unit
  __align__(16) unsigned char answer[16];
  uint64_t kv_full[kRing], kv_empty[kRing];
  uint64_t raw_full[kRing];  // value blocks that have landed and are to be cleaned, in turn
  Unit unit[2];
  int odd[4];       // per unit (by its number mod 4): a value of the cleaned range is not finite
  uint32_t tmem;
  int abort;
  // requested so far, for the wait after an abort
  int loaded, raw_loaded, q_loaded[2];
  int raw[kRing];   // whether a stage's last copy completes on raw_full
};

// Bounded wait of a whole warp; when it runs out the warp's role ends, and
// with it, by sh.abort, every other.
#define TIDE_WAIT(bar, parity)                                                         \
  do {                                                                                 \
    if (!__all_sync(0xffffffffu, ptx::mbar_wait((bar), (parity), &sh.abort))) {        \
      sh.abort = 1;                                                                    \
      raise_error(p.batch.err, TIDE_DEVERR_TIMEOUT);                                   \
      return;                                                                          \
    }                                                                                  \
  } while (0)

// ------------------------------------------------------------------ units
// Units of sequence i, the level of its first one, and its keys.
__device__ __forceinline__ int seq_level(const Params &p, int i, int *count, int *level) {
  const Sequence s = sequence(p.batch, i);
  const unsigned per = 2 * p.tokens;
  *count = s.n > p.few ? (int)((s.n + per - 1) / per) : 0;
  *level = (int)((unsigned)max(s.kv - s.n, 0) / per);
  return s.kv;
}

// The unit of a CTA that has yet to start, which then does not; *more is false
// when there is none.  False when the wait ran out.
__device__ __forceinline__ bool next_unit(const Params &p, Shared &sh, uint32_t *u, uint32_t *asked,
                                          bool *more) {
  if ((threadIdx.x & 31) == 0) {
    ptx::mbar_expect_tx(&sh.taken, 16);
    ptx::clc_try_cancel(sh.answer, &sh.taken);
  }
  __syncwarp();
  if (!__all_sync(0xffffffffu, ptx::mbar_wait(&sh.taken, *asked & 1, &sh.abort))) {
    sh.abort = 1;
    raise_error(p.batch.err, TIDE_DEVERR_TIMEOUT);
    return false;
  }
  ++*asked;
  uint32_t cta = 0;
  *more = ptx::clc_canceled(sh.answer, &cta);
  *u = cta;
  ptx::fence_proxy_async();  // read before the next answer is written
  __syncwarp();
  return true;
}

__device__ void schedule_units(const Params &p, Shared &sh) {
  constexpr unsigned kFull = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int live = live_sequences(p.batch);
  int cnt[kCached], lvl[kCached];
  uint32_t units_in_all = 0;  // of one KV head and split
  int64_t keys_in_all = 0;
  int top = 0;
  {
    unsigned c = 0, low = 0, high = 0;  // (keys: their low and high 16 bits)
    auto add = [&](int i, int *n, int *l) {
      const unsigned kv = (unsigned)seq_level(p, i, n, l);
      c += *n;
      low += kv & 0xffff;
      high += kv >> 16;
      top = max(top, *n + *l);
    };
#pragma unroll
    for (int k = 0; k < kCached; ++k) {
      cnt[k] = lvl[k] = 0;
      if (lane + 32 * k < live) add(lane + 32 * k, &cnt[k], &lvl[k]);
    }
    for (int i = lane + 32 * kCached; i < live; i += 32) {
      int n, l;
      add(i, &n, &l);
    }
    units_in_all = __reduce_add_sync(kFull, c);
    keys_in_all = (int64_t)__reduce_add_sync(kFull, low) + ((int64_t)__reduce_add_sync(kFull, high) << 16);
    top = __reduce_max_sync(kFull, top);
  }
  int s0 = 0, s1 = 0;  // the group: sequences [s0, s1)
  auto units_from = [&](int x) {  // its units of level x and above
    int c = 0;
#pragma unroll
    for (int k = 0; k < kCached; ++k)
      if (lane + 32 * k >= s0 && lane + 32 * k < s1) c += min(max(cnt[k] + lvl[k] - x, 0), cnt[k]);
    for (int i = max(s0 & ~31, 32 * kCached) + lane; i < s1; i += 32) {
      int n = 0, l = 0;
      if (i >= s0) seq_level(p, i, &n, &l);
      c += min(max(n + l - x, 0), n);
    }
    return (int)__reduce_add_sync(kFull, (unsigned)c);
  };
  const uint32_t per_rank = p.hkv * p.splits;
  int base = 0;                      // units (of one KV head and split) before the group
  int total = 0;                     // in the group
  int x = 0, above = 0, upto = 0;    // level, the group's units above it, of it and above
  int top_level = 0;
  if (keys_in_all <= p.group_keys) {  // one group: all of them
    s1 = live;
    total = (int)units_in_all;
    x = top_level = top;
  }
  uint32_t asked = 0;
  bool more = true;  // this CTA has a unit
  uint32_t u = blockIdx.x;
  for (uint32_t n = 0;; ++n) {
    const int slot = n & 1;
    // every warp has taken up the unit before: time for another one (sooner,
    // and at the end one CTA would hold what another could run)
    if (n > 0 && !p.take_over) more = false;
    if (n > 0 && more) {
      TIDE_WAIT(&sh.u_empty[slot ^ 1], ((n - 1) >> 1) & 1);
      if (!next_unit(p, sh, &u, &asked, &more)) return;
    }
    // a CTA without a unit takes over what else there is without one
    while (more && u / per_rank >= units_in_all) {
      if (!p.take_over) more = false;
      else if (!next_unit(p, sh, &u, &asked, &more)) return;
    }
    const int rank = (int)(u / per_rank);
    if (rank < base) s1 = total = 0, base = 0;  // (should they ever come out of order)
    while (rank - base >= total && s1 < live) {  // the next group
      base += total;
      s0 = s1;
      int64_t keys = 0;
      int most = 0;
      for (;;) {
        const int i = s1 + lane;
        const int mine = i < live ? sequence(p.batch, i).kv : 0;
        int64_t sum = mine;
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
          const int64_t y = __shfl_up_sync(kFull, sum, w);
          if (lane >= w) sum += y;
        }
        const bool in = i < live && (keys + sum <= p.group_keys / 4 * 3 || i == s0);
        const int many = __popc(__ballot_sync(kFull, in));
        if (in) {
          int c, l;
          seq_level(p, i, &c, &l);
          most = max(most, c + l);
        }
        keys += __shfl_sync(kFull, sum, 31);
        s1 += many;
        if (many < 32) break;
      }
      x = top_level = __reduce_max_sync(kFull, most);
      above = upto = 0;
      total = units_from(0);
    }
    Unit w{};
    if (more && rank < (int)units_in_all) {
      const int in_group = rank - base;
      if (in_group < above) x = top_level, above = upto = 0;
      if (in_group >= upto) {  // units_from(lo) > in_group >= units_from(hi)
        int lo = 0, hi = x;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (units_from(mid) > in_group) lo = mid;
          else hi = mid;
        }
        x = lo;
        upto = units_from(lo);
        above = units_from(hi);
      }
      int r = in_group - above;  // the r-th sequence of the group with a unit of level x
      int seq = -1, level = 0;
#pragma unroll
      for (int k = 0; k < kCached; ++k) {
        const int i = lane + 32 * k;
        const bool has = i >= s0 && i < s1 && lvl[k] <= x && x < lvl[k] + cnt[k];
        const unsigned who = __ballot_sync(kFull, has);
        if (seq < 0) {
          if (r < __popc(who)) {
            const bool me = has && __popc(who & ((1u << lane) - 1)) == r;
            const int src = __ffs(__ballot_sync(kFull, me)) - 1;
            seq = src + 32 * k;
            level = __shfl_sync(kFull, lvl[k], src);
          } else {
            r -= __popc(who);
          }
        }
      }
      for (int b = max(s0 & ~31, 32 * kCached); seq < 0 && b < s1; b += 32) {
        int c = 0, l = 0;
        if (b + lane >= s0 && b + lane < s1) seq_level(p, b + lane, &c, &l);
        const bool has = l <= x && x < l + c;
        const unsigned who = __ballot_sync(kFull, has);
        if (r < __popc(who)) {
          const bool me = has && __popc(who & ((1u << lane) - 1)) == r;
          const int src = __ffs(__ballot_sync(kFull, me)) - 1;
          seq = src + b;
          level = __shfl_sync(kFull, l, src);
        } else {
          r -= __popc(who);
        }
      }
      const Sequence s = sequence(p.batch, seq);
      const int at = (x - level) * 2 * p.tokens;
      const int rest = (int)(u % per_rank);
      w.valid = 1;
      w.row0 = s.row0 + at;
      w.n = min(2 * p.tokens, s.n - at);
      w.pos0 = s.kv - s.n + at;
      w.kvh = rest / p.splits;
      w.split = rest % p.splits;
      w.req = s.req;
      w.key0 = s.row0;
      w.b0 = w.split * p.split_blocks;
      w.b1 = w.b0 + p.split_blocks;
    }
    if (lane == 0) {
      sh.unit[slot] = w;
      ptx::mbar_arrive(&sh.u_full[slot]);
    }
    __syncwarp();
    if (!w.valid) return;
  }
}

// The next unit of a warp's role; its slot is free again once every warp has
// read it.
#define TIDE_NEXT_UNIT(u, n)                                          \
  TIDE_WAIT(&sh.u_full[(n) & 1], ((n) >> 1) & 1);                     \
  const Unit u = sh.unit[(n) & 1];                                    \
  __syncwarp();                                                       \
  if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(&sh.u_empty[(n) & 1]); \
  if (!u.valid) break

// ---------------------------------------------------------------- loading
template <int D, bool PAGED>
__device__ void load_units(const Params &p, Shared &sh, unsigned char *q_smem,
                           unsigned char *ring, const CUtensorMap *mq, const CUtensorMap *mk,
                           const CUtensorMap *mv) {
  using S = Shape<D>;
  const int lane = threadIdx.x & 31;
  uint32_t c = 0;         // K and V blocks requested so far
  uint32_t raw = 0;       // of them to be cleaned
  uint32_t nq[2] = {0, 0};
  const int page = 1 << p.src.page_shift;
  const int box = min(page, kKeys);           // rows of a copy
  const int boxes = kKeys / box;              // copies a column group takes
  const uint32_t q_bytes = (uint32_t)(p.tokens * p.group) * 128u * S::kHalves;
  for (uint32_t n = 0;; ++n) {
    TIDE_NEXT_UNIT(u, n);
    const int ends[2] = {tile_end(u, p.tokens, 0), tile_end(u, p.tokens, 1)};
    const int end = max(ends[0], ends[1]);
    if (end <= u.b0) continue;
    const int sees = u.pos0 + u.n;
    // the queries into L2 while their place in shared memory is still in use
    if (lane < 2 * S::kHalves && ends[lane / S::kHalves] > u.b0)
      ptx::tma_prefetch_3d(mq, lane % S::kHalves * 64, u.kvh * p.group,
                           u.row0 + lane / S::kHalves * p.tokens);
    // the pages of a block, one per lane; the next block's are read ahead
    auto page_of = [&](int j) {
      int row = -1;
      if (PAGED && lane < boxes && j < end && j * kKeys + lane * box < sees) {
        const int at = j * kKeys + lane * box;
        const int pg = __ldg(p.src.tables + u.req * p.src.max_pages + (at >> p.src.page_shift));
        const bool real = pg >= 0 && pg < p.src.n_pages;
        if (!real) raise_error(p.batch.err, TIDE_DEVERR_POSITION);
        // a row past the cache's last reads as zeros
        row = ((real ? pg : p.src.n_pages) * p.hkv + (real ? u.kvh : 0)) * page + (at & (page - 1));
      }
      return row;
    };
    int row = page_of(u.b0);
    for (int j = u.b0; j < end; ++j) {
      const int next = page_of(j + 1);
      const int count = PAGED ? (min(kKeys, sees - j * kKeys) + box - 1) / box : 1;  // copies
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t stage = c % S::kStages, lap = c / S::kStages;
        if (lap >= 1) TIDE_WAIT(&sh.kv_empty[stage], (lap + 1) & 1);
        unsigned char *dst = ring + stage * S::kBlock;
        const CUtensorMap *m = kv ? mv : mk;
        int from, to;
        const bool dirty = kv && cleaned_rows(u, sees, j, &from, &to);
        uint64_t *full = dirty ? &sh.raw_full[raw % S::kStages] : &sh.kv_full[stage];
        raw += dirty;
        if (lane == 0) {
          ptx::mbar_expect_tx(full, PAGED ? (uint32_t)(count * box) * 128u * S::kHalves : S::kBlock);
          sh.raw[stage] = dirty;
          sh.loaded = (int)c + 1;
          sh.raw_loaded = (int)raw;
        }
        __syncwarp();
        if (PAGED) {
          const int r = lane / S::kHalves, h = lane % S::kHalves;
          const int src = __shfl_sync(0xffffffffu, row, r);
          if (r < count) ptx::tma_load_2d(dst + h * S::kHalf + r * box * 128, m, full, h * 64, src);
        } else if (lane < S::kHalves) {
          ptx::tma_load_3d(dst + lane * S::kHalf, m, full, lane * 64, u.kvh, u.key0 + j * kKeys);
        }
        ++c;
        // The queries go between the first keys and values: the products wait
        // for Q before they free what the values need.
        if (j == u.b0 && kv == 0)
          for (int t = 0; t < 2; ++t) {
            if (ends[t] <= u.b0) continue;
            if (nq[t] >= 1) TIDE_WAIT(&sh.q_empty[t], (nq[t] + 1) & 1);
            ++nq[t];
            if (lane == 0) {
              sh.q_loaded[t] = (int)nq[t];
              ptx::mbar_expect_tx(&sh.q_full[t], q_bytes);
            }
            __syncwarp();
            if (lane < S::kHalves)
              ptx::tma_load_3d(q_smem + t * S::kQ + lane * S::kQHalf, mq, &sh.q_full[t], lane * 64,
                               u.kvh * p.group, u.row0 + t * p.tokens);
          }
      }
      row = next;
    }
  }
}

// --------------------------------------------------------------- products
// The products of both tiles, in turn: per block and tile the value product,
// as soon as P is written, then the scores of the next block.  The last tile
// that reads a block frees it.  What the warp does between two products is on
// the chain of both tiles, so it is kept short.  The whole warp walks through
// the schedule with values that are the same in every lane, and one elected
// lane issues: the operands of tcgen05.mma live in uniform registers, and
// per-lane values would be moved there one by one (107 cycles a product
// instead of 80).  uniform() tells the compiler: a reduction over the warp is
// a uniform value.
__device__ __forceinline__ int uniform(int x) {
  return (int)__reduce_or_sync(0xffffffffu, (unsigned)x);
}

template <typename T, int D>
__device__ void issue_products(const Params &p, Shared &sh, uint32_t q_smem, uint32_t ring,
                               uint32_t tmem) {
  using S = Shape<D>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kPvDesc = ptx::f16_idesc(kBf16, kRows, D) | ptx::kIdescMnMajorB;
  constexpr uint32_t kBlockDesc = S::kBlock >> 4;
  tmem = (uint32_t)uniform((int)tmem);
  const uint64_t q_desc = ptx::sw128_kmajor_desc((uint32_t)uniform((int)q_smem));
  const uint64_t k_desc = ptx::sw128_kmajor_desc((uint32_t)uniform((int)ring));
  const uint64_t v_desc = ptx::sw128_mnmajor_desc((uint32_t)uniform((int)ring), S::kHalf);
  uint32_t stage = 0, lap = 0;  // of the next K block
  uint32_t nq = 0, np = 0;      // bit t: phases of tile t's barriers
  for (uint32_t n = 0;; ++n) {
    TIDE_NEXT_UNIT(u, n);
    const int b0 = uniform(u.b0);
    const int end0 = uniform(tile_end(u, p.tokens, 0)), end1 = uniform(tile_end(u, p.tokens, 1));
    const int sees0 = uniform(tile_sees(u, p.tokens, 0)), sees1 = uniform(tile_sees(u, p.tokens, 1));
    const int end = max(end0, end1);
    if (end <= b0) continue;
    // S_t = Q_t K_j^T over the keys that the tile sees, rounded up to 16
    auto scores = [&](int t, int j, uint32_t k_stage) {
      const int keys = min(kKeys, (t ? sees1 : sees0) - j * kKeys);
      const uint32_t idesc = ptx::f16_idesc(kBf16, kRows, 0) | (uint32_t)((keys + 15) / 16 * 2) << 17;
      const uint64_t a = q_desc + t * (S::kQ >> 4), b = k_desc + k_stage * kBlockDesc;
      if (ptx::elect_one()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          ptx::mma_f16_ss(tmem + t * 256, a + (k / 4) * (S::kQHalf >> 4) + (k % 4) * 2,
                          b + (k / 4) * (S::kHalf >> 4) + (k % 4) * 2, idesc, k > 0);
        ptx::mma_commit(&sh.s_full[t]);
        if (j + 1 == (t ? end1 : end0)) ptx::mma_commit(&sh.q_empty[t]);
        if (t == 1 || j >= end1) ptx::mma_commit(&sh.kv_empty[k_stage]);
      }
      __syncwarp();
    };
    TIDE_WAIT(&sh.kv_full[stage], lap & 1);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (b0 >= (t ? end1 : end0)) continue;
      TIDE_WAIT(&sh.q_full[t], (nq >> t) & 1);
      nq ^= 1u << t;
      ptx::tc_fence_after();
      scores(t, b0, stage);
    }
    for (int j = b0; j < end; ++j) {
      uint32_t v_stage = stage + 1, v_lap = lap;
      if (v_stage == S::kStages) v_stage = 0, ++v_lap;
      stage = v_stage + 1, lap = v_lap;
      if (stage == S::kStages) stage = 0, ++lap;
      TIDE_WAIT(&sh.kv_full[v_stage], v_lap & 1);
      if (j + 1 < end) TIDE_WAIT(&sh.kv_full[stage], lap & 1);  // K of the next block
      const uint64_t vb = v_desc + v_stage * kBlockDesc;
      const uint32_t more = j > b0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int end_t = t ? end1 : end0;
        if (j >= end_t) continue;
        // O_t += P_t V_j, 16 keys at a time: three quarters of the block as
        // soon as they are there, then the rest
        const int steps = (min(kKeys, (t ? sees1 : sees0) - j * kKeys) + 15) / 16;
        const uint32_t o_col = tmem + t * 256 + kKeys, p_col = tmem + t * 256 + kKeys / 2;
        TIDE_WAIT(&sh.p_full[t][0], (np >> t) & 1);
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
#pragma unroll
          for (int k = 0; k < 6; ++k)
            if (k < steps)
              ptx::mma_f16_ts(o_col, p_col + k * 8, vb + k * (2048 >> 4), kPvDesc, k ? 1u : more);
        }
        __syncwarp();
        TIDE_WAIT(&sh.p_full[t][1], (np >> t) & 1);
        np ^= 1u << t;
        ptx::tc_fence_after();
        const bool last = j + 1 == end_t;
        if (ptx::elect_one()) {
#pragma unroll
          for (int k = 6; k < 8; ++k)
            if (k < steps) ptx::mma_f16_ts(o_col, p_col + k * 8, vb + k * (2048 >> 4), kPvDesc, 1u);
          if (last) ptx::mma_commit(&sh.o_full[t]);
          if (t == 1 || j >= end1) ptx::mma_commit(&sh.kv_empty[v_stage]);
        }
        __syncwarp();
        if (!last) scores(t, j + 1, stage);
      }
    }
  }
}

// ---------------------------------------------------------------- cleaning
template <typename T>
__device__ __forceinline__ bool odd_value(uint32_t bits16) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (bits16 & kExp) == kExp;
}

template <typename P2>
__device__ __forceinline__ P2 make_pair() {  // two zeros
  P2 r;
  *reinterpret_cast<uint32_t *>(&r) = 0u;
  return r;
}

template <typename T, int D>
__device__ void clean_values(const Params &p, Shared &sh, unsigned char *ring) {
  using S = Shape<D>;
  using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  constexpr int kBatch = 4;  // vectors in flight per lane
  const int lane = threadIdx.x & 31;
  uint32_t c0 = 0, raw = 0;  // ring count of the unit's first K block, cleaned blocks
  for (uint32_t n = 0;; ++n) {
    TIDE_NEXT_UNIT(u, n);
    const int end = max(tile_end(u, p.tokens, 0), tile_end(u, p.tokens, 1));
    if (lane == 0) sh.odd[n & 3] = 0;
    __syncwarp();
    if (end <= u.b0) continue;
    const int sees = u.pos0 + u.n;
    // (only the last blocks hold positions past the first token's own)
    for (int j = max(u.b0, (u.pos0 + 1) / kKeys); j < end; ++j) {
      int from, to;
      if (!cleaned_rows(u, sees, j, &from, &to)) continue;
      const uint32_t stage = (c0 + 2 * (j - u.b0) + 1) % S::kStages;
      TIDE_WAIT(&sh.raw_full[raw % S::kStages], (raw / S::kStages) & 1);
      ++raw;
      unsigned char *v = ring + stage * S::kBlock;
      const int seen = min(kKeys, sees - j * kKeys);  // rows that some token sees
      // a row is 8 16-byte vectors in each column group; a swizzle moves them
      // within their 128 bytes only
      auto vec = [&](int e) {
        return reinterpret_cast<uint4 *>(v + (e / 8 % S::kHalves) * S::kHalf +
                                         e / (8 * S::kHalves) * 128 + e % 8 * 16);
      };
      constexpr int kRowVecs = 8 * S::kHalves;
      for (int e = max(seen, from) * kRowVecs + lane; e < to * kRowVecs; e += 32)
        *vec(e) = make_uint4(0, 0, 0, 0);
      // x * 0 is NaN for a NaN and for an infinity: one instruction for two
      // values (the warp that cleans shares its scheduler with two softmax
      // warps, and the products wait for the block)
      Pair zero, acc;
      zero = acc = make_pair<Pair>();
      for (int e = from * kRowVecs + lane; e < seen * kRowVecs; e += 32 * kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) x[i] = *vec(min(e + 32 * i, seen * kRowVecs - 1));
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const Pair *w = reinterpret_cast<const Pair *>(&x[i]);
#pragma unroll
          for (int h = 0; h < 4; ++h) acc = __hfma2(w[h], zero, acc);
        }
      }
      const bool odd = (*reinterpret_cast<uint32_t *>(&acc) & 0x7FFF7FFFu) != 0;
      if (__any_sync(0xffffffffu, odd)) {
        for (int e = from * kRowVecs + lane; e < seen * kRowVecs; e += 32) {
          uint32_t *w = reinterpret_cast<uint32_t *>(vec(e));
          for (int h = 0; h < 4; ++h) {
            if (odd_value<T>(w[h])) w[h] &= 0xFFFF0000u;
            if (odd_value<T>(w[h] >> 16)) w[h] &= 0x0000FFFFu;
          }
        }
        if (lane == 0) sh.odd[n & 3] = 1;
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.kv_full[stage]);
    }
    c0 += 2 * (end - u.b0);
  }
}

// ----------------------------------------------------------------- softmax
// The values that the cleaner zeroed in the positions that this row sees, for
// the columns [d0, d0 + 32): weight > 0 times a NaN or infinity is itself.
template <typename T, int D, bool PAGED>
__device__ __forceinline__ void add_odd_values(const Params &p, const Unit &u, int first, int last,
                                               int d0, float *o) {
  const T *v = static_cast<const T *>(p.src.v);
  const int page = 1 << p.src.page_shift;
  for (int pos = first; pos < last; ++pos) {
    int64_t at;
    if (PAGED) {
      const int pg = __ldg(p.src.tables + u.req * p.src.max_pages + (pos >> p.src.page_shift));
      if (pg < 0 || pg >= p.src.n_pages) continue;
      at = (((int64_t)pg * p.hkv + u.kvh) * page + (pos & (page - 1))) * D;
    } else {
      at = (int64_t)(u.key0 + pos) * p.src.row_stride + (int64_t)u.kvh * D;
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const float x = Elem<T>::to_f(v[at + d0 + e]);
      if (!isfinite(x)) o[e] += x;
    }
  }
}

// Rows of a warp to global memory, N 16-byte vectors of each of its 32 rows at
// a time, row r in lane r: over shared memory, so that N lanes write a row's
// bytes side by side (a lane that wrote its own row would touch 32 lines an
// instruction).  The places are found once, and the loads from shared memory
// are all issued before the first store (one after the other, behind stores
// that might have been to the same place, they made a unit's end 4700 cycles
// long).
template <int N>
struct RowStore {
  static constexpr int kRowsAtOnce = 32 / N;
  unsigned char *to[N];
  int lane;

  // at: this lane's row in global memory, or NULL
  __device__ __forceinline__ RowStore(unsigned char *at, int lane) : lane(lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned char *a = reinterpret_cast<unsigned char *>(__shfl_sync(
          0xffffffffu, reinterpret_cast<unsigned long long>(at), i * kRowsAtOnce + lane / N));
      to[i] = a ? a + lane % N * 16 : nullptr;
    }
  }
  // w to the bytes from `offset` on of each row
  __device__ __forceinline__ void operator()(uint32_t staging, const uint32_t *w, int offset) const {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; ++i)
      ptx::sts128(staging + lane * 128 + ((i ^ (lane & 7)) << 4), w + 4 * i);
    __syncwarp();
    uint4 x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * kRowsAtOnce + lane / N;
      x[i] = ptx::lds128(staging + r * 128 + ((lane % N ^ (r & 7)) << 4));
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (to[i]) *reinterpret_cast<uint4 *>(to[i] + offset) = x[i];
  }
};

// Weights of 32 scores, their sums, and their 16-bit form to tensor memory.
// MORE: also the largest of the first MORE scores, in the shadow of the
// exponentials (16 lanes a cycle per SM, eight cycles for a warp's).
template <typename T, int MORE>
__device__ __forceinline__ void weigh_quarter(const float *s, uint64_t qs2, uint64_t mq2,
                                              uint64_t (&sum)[2], uint32_t p_col, float (&mx)[2]) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float a, b;
    if (MORE) mx[i & 1] = max3(mx[i & 1], s[2 * i], s[2 * i + 1]);
    if (MORE > 32) mx[i & 1] = max3(mx[i & 1], s[32 + 2 * i], s[32 + 2 * i + 1]);
    unpair(fma2(pair(s[2 * i], s[2 * i + 1]), qs2, mq2), &a, &b);
    a = ex2(a);
    b = ex2(b);
    sum[i & 1] = add2(sum[i & 1], pair(a, b));
    w[i] = pack_weights<T>(a, b);
  }
  ptx::tmem_st16(p_col, w);
}

template <typename T, int D, bool PAGED>
__device__ void softmax_tile(const Params &p, Shared &sh, int t, uint32_t tmem,
                             uint32_t stage, const CUtensorMap *mo) {
  constexpr unsigned kFull = 0xffffffffu;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3;
  const int r = warp * 32 + lane;                 // row of the tile
  const int tok = r / p.group, head = r % p.group;
  const uint32_t s_col = tmem + ((uint32_t)(warp * 32) << 16) + t * 256;
  const uint32_t p_col = s_col + kKeys / 2, o_col = s_col + kKeys;
  const float slack = kSlack / p.qs;
  uint32_t ns = 0, no = 0;  // blocks and units so far
  for (uint32_t n = 0;; ++n) {
    TIDE_NEXT_UNIT(u, n);
    const int tokens = tile_tokens(u, p.tokens, t);
    if (!tokens) continue;
    const int end = tile_end(u, p.tokens, t);
    const bool valid = tok < tokens;
    const bool busy = __any_sync(kFull, valid);  // (the first token's warps always are)
    const int last = tile_sees(u, p.tokens, t);
    // keys this row sees (a row that is not there: as many as the last one)
    const int sees = valid ? u.pos0 + t * p.tokens + tok + 1 : last;
    const int64_t row = u.row0 + t * p.tokens + tok;
    float m = -INFINITY, l = 0.f;
    if (p.zero_keys && valid) {  // keys of score 0 whose values add nothing
      const int z = max(__ldg(p.zero_keys + row), 0);
      if (z) m = 0.f;
      l = (float)z * kLifted<T>;
    }
    for (int j = u.b0; j < end; ++j, ++ns) {
      TIDE_WAIT(&sh.s_full[t], ns & 1);
      // The commit behind S_j follows the products of block j - 1 in the same
      // stream: O is complete up to that block.
      if (!busy) {
        if (lane == 0) {
          ptx::mbar_arrive(&sh.p_full[t][0]);
          ptx::mbar_arrive(&sh.p_full[t][1]);
        }
        continue;
      }
      ptx::tc_fence_after();
      const int lim = sees - j * kKeys;        // keys from here on: masked, or not computed
      uint32_t sr[kKeys];
      float *s = reinterpret_cast<float *>(sr);
#pragma unroll
      for (int q = 0; q < 4; ++q) ptx::tmem_ld32_async(s_col + q * kQuarter, sr + q * kQuarter);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < 4; ++q) ptx::tmem_landed(sr + q * kQuarter);
      if (__any_sync(kFull, lim < kKeys)) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) s[i] = i < lim ? s[i] : -INFINITY;
      }
      // Weights of three quarters against the maximum as it was, and the
      // maximum beside them: a block rarely has a score more than kSlack above
      // it, and if it has they are weighed once more.  (With the maximum first
      // each block's chain was 250 of 3350 cycles longer.)
      uint64_t sum[2], qs2, mq2;
      float mx[2];
      auto weigh = [&] {  // S is in registers: P takes its upper half
        const float mq = (m == -INFINITY ? 0.f : m * p.qs) - kLift<T>;
        qs2 = pair(p.qs, p.qs), mq2 = pair(-mq, -mq);
        sum[0] = sum[1] = 0;
        mx[0] = mx[1] = -INFINITY;
        weigh_quarter<T, 32>(s, qs2, mq2, sum, p_col, mx);
        weigh_quarter<T, 32>(s + 32, qs2, mq2, sum, p_col + 16, mx);
        weigh_quarter<T, 64>(s + 64, qs2, mq2, sum, p_col + 32, mx);
      };
      if (j == u.b0) {  // nothing in O yet
        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kKeys; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = max3(x[q], s[i + 2 * q], s[i + 2 * q + 1]);
        const float top = fmaxf(max3(x[0], x[1], x[2]), x[3]);
        if (top > m) {
          l *= ex2((m - top) * p.qs);
          m = top;
        }
      }
#pragma unroll 1
      for (;;) {
        weigh();
        const float top = fmaxf(mx[0], mx[1]);
        const bool raise = top > m + slack;  // (never in a unit's first block)
        if (!__any_sync(kFull, raise)) break;
        const float a = raise ? ex2((m - top) * p.qs) : 1.f;
        if (raise) m = top;
        l *= a;
#pragma unroll 1
        for (int q = 0; q < D; q += 16) {
          uint32_t o[16];
          ptx::tmem_ld16_async(o_col + q, o);
          ptx::tmem_wait_ld();
          ptx::tmem_landed16(o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
          ptx::tmem_st16(o_col + q, o);
        }
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.p_full[t][0]);
      weigh_quarter<T, 0>(s + 96, qs2, mq2, sum, p_col + 48, mx);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.p_full[t][1]);
      float la, lb;
      unpair(add2(sum[0], sum[1]), &la, &lb);
      l += la + lb;
    }
    const bool some = end > u.b0;
    const int64_t at = row * p.hq + u.kvh * p.group + head;
    const bool nothing = !some || l == 0.f;
    const float inv = nothing ? 0.f : 1.f / l;
    const int64_t part = (int64_t)u.split * p.batch.n_tokens * p.hq + at;
    if (p.splits > 1 && valid) p.part_ml[part] = make_float2(m * p.qs, l);
    if (some) {
      TIDE_WAIT(&sh.o_full[t], no & 1);
      ++no;
      ptx::tc_fence_after();
    }
    if (!busy) continue;
    const bool odd = some && sh.odd[n & 3];
    const int first = max(u.pos0 + 1, u.b0 * kKeys);
    const int stop = valid ? min(sees, min(end * kKeys, last)) : first;
    auto output = [&](int q, uint32_t(&o)[32]) {
      if (some) {
        ptx::tmem_ld32_async(o_col + q, o);
        ptx::tmem_wait_ld();
        ptx::tmem_landed(o);
      }
      if (odd) add_odd_values<T, D, PAGED>(p, u, first, stop, q, reinterpret_cast<float *>(o));
    };
    // (The addresses below are worked out here: kept over the loop above they
    // would cost it registers.)
    int me = lane;
    uint32_t staging = stage;
    asm volatile("" : "+r"(me), "+r"(staging));
    // copies out of the staging that the unit before left in flight
    if (lane == 0) ptx::bulk_wait_read(0);
    __syncwarp();
    if (p.splits > 1) {
      if (!some) continue;  // (a sum of 0: its output is not read)
      const RowStore<8> store(valid ? reinterpret_cast<unsigned char *>(p.part_o + part * D) : nullptr,
                              me);
#pragma unroll 1
      for (int q = 0; q < D; q += 32) {
        uint32_t o[32];
        output(q, o);
        store(staging, o, q * 4);
      }
    } else {
      // When all 32 rows are there, and they are whole tokens' heads, or heads
      // of one token: copies of 32 columns, two of them in flight, from 64-byte
      // rows swizzled as the copy expects.
      const bool box = p.boxes && __all_sync(kFull, valid);
      const int tok0 = __shfl_sync(kFull, (int)row, 0), head0 = __shfl_sync(kFull, u.kvh * p.group + head, 0);
      const RowStore<4> store(
          valid ? reinterpret_cast<unsigned char *>(static_cast<T *>(p.out) + at * D) : nullptr, me);
#pragma unroll 1
      for (int q = 0; q < D; q += 32) {
        uint32_t o[32], w[16];
        output(q, o);
        const float *f = reinterpret_cast<const float *>(o);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = nothing ? 0u : pack2<T>(f[2 * i] * inv, f[2 * i + 1] * inv);
        if (box) {
          const uint32_t half = (q & 32) * 64;
          if (lane == 0) ptx::bulk_wait_read(1);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ptx::sts128(staging + half + me * 64 + ((i ^ ((me >> 1) & 3)) << 4), w + 4 * i);
          ptx::fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            ptx::tma_store_3d(mo, staging + half, q, head0, tok0);
            ptx::bulk_commit();
          }
        } else {
          store(staging, w, q * 2);
        }
      }
    }
    ptx::tc_fence_before();
  }
}

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
    tile_attention_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap mq,
                          const __grid_constant__ CUtensorMap mk,
                          const __grid_constant__ CUtensorMap mv,
                          const __grid_constant__ CUtensorMap mo) {
  using S = Shape<D>;
  extern __shared__ unsigned char dyn[];
  __shared__ Shared sh;
  unsigned char *base = dyn + ((1024u - (ptx::smem_u32(dyn) & 1023u)) & 1023u);
  unsigned char *q_smem = base, *ring = base + 2 * S::kQ;
  unsigned char *staging = ring + S::kStages * S::kBlock;
  const int warp = threadIdx.x >> 5;
  if (p.needed) {  // (its set-up costs a round of CTAs some 9 us)
    ptx::grid_dependency_wait();
    if (__ldcg(p.needed) == 0) return;
  }
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&sh.q_full[t], 1);
      ptx::mbar_init(&sh.q_empty[t], 1);
      ptx::mbar_init(&sh.s_full[t], 1);
      for (int b = 0; b < 2; ++b) ptx::mbar_init(&sh.p_full[t][b], 4);
      ptx::mbar_init(&sh.o_full[t], 1);
      ptx::mbar_init(&sh.u_full[t], 1);
      ptx::mbar_init(&sh.u_empty[t], kReaders);
    }
    for (int i = 0; i < S::kStages; ++i) {
      ptx::mbar_init(&sh.kv_full[i], 1);
      ptx::mbar_init(&sh.kv_empty[i], 1);
      ptx::mbar_init(&sh.raw_full[i], 1);
      sh.raw[i] = 0;
    }
    ptx::mbar_init(&sh.drain, 1);
    ptx::mbar_init(&sh.taken, 1);
    ptx::fence_mbar_init();
    sh.abort = 0;
    sh.loaded = sh.raw_loaded = sh.q_loaded[0] = sh.q_loaded[1] = 0;
  }
  if (warp == 10) {
    ptx::tmem_alloc(&sh.tmem, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // Up to here this overlaps the kernel before.  (Over the few-rows kernel of
  // the same call, which waits before it lets this one start, there is nothing
  // more to wait for.)
  if (!p.behind_few) ptx::grid_dependency_wait();
  if (threadIdx.x == 0) ptx::grid_dependents_launch();

  // Registers move to the softmax warps: 256 * 208 + 128 * 88 = 384 * 168, what
  // the block was launched with.
  if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp < 8) {
    softmax_tile<T, D, PAGED>(p, sh, warp >> 2, tmem, ptx::smem_u32(staging + warp * 4096), &mo);
    if ((threadIdx.x & 31) == 0) ptx::bulk_wait_all();
  } else if (warp == 8) {
    schedule_units(p, sh);
  } else if (warp == 9) {
    load_units<D, PAGED>(p, sh, q_smem, ring, &mq, &mk, &mv);
  } else if (warp == 10) {
    issue_products<T, D>(p, sh, ptx::smem_u32(q_smem), ptx::smem_u32(ring), tmem);
    __syncwarp();
    // every product done before its memory goes (after an abort too; bounded)
    if (ptx::elect_one()) {
      volatile int none = 0;
      ptx::mma_commit(&sh.drain);
      ptx::mbar_wait(&sh.drain, 0, &none);
    }
    __syncwarp();
  } else {
    clean_values<T, D>(p, sh, ring);
  }
  __syncthreads();
  if (sh.abort && threadIdx.x == 0) {  // copies may still be landing: wait for them (bounded)
    volatile int none = 0;
    for (int c = max(0, sh.loaded - S::kStages); c < sh.loaded; ++c)
      if (!sh.raw[c % S::kStages])
        ptx::mbar_wait(&sh.kv_full[c % S::kStages], (c / S::kStages) & 1, &none);
    for (int c = max(0, sh.raw_loaded - S::kStages); c < sh.raw_loaded; ++c)
      ptx::mbar_wait(&sh.raw_full[c % S::kStages], (c / S::kStages) & 1, &none);
    for (int t = 0; t < 2; ++t)
      if (sh.q_loaded[t]) ptx::mbar_wait(&sh.q_full[t], (sh.q_loaded[t] - 1) & 1, &none);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 10) ptx::tmem_dealloc(tmem, 512);
  // what comes after this kernel comes after the few-rows kernel too
  if (p.behind_few && threadIdx.x == 0) ptx::grid_dependency_wait();
}

// --------------------------------------------------------- few rows a head
// Sequences with few rows (tokens times the query heads of a KV head): a
// decode step, a few drafted tokens.  Such a unit reads 4 D bytes per key and
// does 4 D flops per key and row, so it is bound by HBM, and the 128-row tiles
// above would leave it to one chain of products and exponentials per SM.  A
// CTA takes 8 NT rows; a sequence with more, up to twice as many, has two, which
// share their keys through L2.  A warp is on its own: it walks over
// every fourth group of 16 keys of its CTA's share, with its own ring of TMA
// copies (8 KB a group, three in flight) and its own running maxima, sums and
// outputs, and the four meet once at the end.  No barrier but the ring's.
//   S^T[16 x 8 NT] = K Q^T   mma.sync m16n8k16, K by ldmatrix from the swizzled
//                            copy, Q in registers;
//   O^T[D x 8 NT] += V^T P^T V by transposing ldmatrix, P from the registers
//                            that held S, each 8 x 8 of it transposed.
// The rows are the narrow side of the products, so they are padded to 8 only:
// these products run at some 32 cycles each per SM partition (tcgen05 has
// nothing to give here, its rows would be padding), which with rows padded to
// 16 was more than the time that the keys of 32 rows take to arrive.
// Measured, 32 query heads on 8 KV heads of 128: 192 requests of 512 to 1535
// keys 121 us, 6.7 TB/s; three of 9000 to 40000 keys 48 us, of which some
// 12 are the start, the end and the join; one of 1000 keys 7.8 us.
constexpr int kFewWarps = 4;
constexpr int kFewStages = 3;
constexpr int kFewKeys = 16;

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
struct FewParams {
  RaggedBatch batch;
  KeySource src;
  const void *q;
  int64_t q_stride;
  void *out;
  float *part_o;    // [splits, n_seqs, few, hq, D] (splits > 1)
  float2 *part_ml;  // [splits, n_seqs, few, hq]: maximum (scaled, base 2), sum
  int hq, hkv, group;
  int few;         // tokens a sequence may have
  int tokens;      // of a CTA: 8 NT / group
  int pieces;      // pieces of up to `tokens` tokens that the sequences may have
  int splits;
  int split_keys;  // keys of a split, a multiple of 16
  float qs;
};

template <int D>
struct Few {
  static constexpr uint32_t kHalf = kFewKeys * 128;              // a 128-byte column group of 16 keys
  static constexpr uint32_t kSide = kHalf * (D / 64);            // K or V of 16 keys
  static constexpr uint32_t kRing = kFewStages * 2 * kSide;      // of a warp
  static constexpr uint32_t kSmem = kFewWarps * kRing + 1024;    // + alignment
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kFewWarps, NT <= 2 ? 3 : 2)
    few_rows_kernel(const __grid_constant__ FewParams p, const __grid_constant__ CUtensorMap mk,
                    const __grid_constant__ CUtensorMap mv) {
  using F = Few<D>;
  constexpr unsigned kFull = 0xffffffffu;
  constexpr int kHalves = D / 64, kRowsMost = 8 * NT;
  extern __shared__ unsigned char dyn[];
  __shared__ uint64_t full[kFewWarps][kFewStages];
  __shared__ float s_m[kFewWarps][kRowsMost], s_l[kFewWarps][kRowsMost];
  __shared__ int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&mk);
    ptx::prefetch_tmap(&mv);
    for (int w = 0; w < kFewWarps; ++w)
      for (int i = 0; i < kFewStages; ++i) ptx::mbar_init(&full[w][i], 1);
    ptx::fence_mbar_init();
    s_abort = 0;
  }
  ptx::grid_dependency_wait();  // up to here this overlaps the kernel before
  ptx::grid_dependents_launch();
  const int split = (int)(blockIdx.x % p.splits);
  const int64_t unit = blockIdx.x / p.splits;
  const int kvh = (int)(unit % p.hkv);
  const int live = live_sequences(p.batch);
  int seq = (int)(unit / p.hkv), tok0 = 0;  // this CTA's tokens from tok0 on
  if (p.few > p.tokens) {
    // pieces of the sequences, counted in their order, 32 sequences at a time
    int rest = seq, found = -1;
    for (int b = 0; b < live && found < 0; b += 32) {
      int mine = 0;
      if (b + lane < live) {
        int row, end;
        const bool good = sequence_bounds(p.batch, b + lane, &row, &end);
        // (one that has no piece here, and with that no CTA to flag it)
        if (!good) raise_error(p.batch.err, TIDE_DEVERR_POSITION);
        const int n = good ? end - row : 0;
        mine = n <= p.few ? (n + p.tokens - 1) / p.tokens : 0;
      }
      int upto = mine;
#pragma unroll
      for (int w = 1; w < 32; w *= 2) {
        const int x = __shfl_up_sync(kFull, upto, w);
        if (lane >= w) upto += x;
      }
      const unsigned past = __ballot_sync(kFull, upto > rest);
      if (past) {
        const int at = __ffs(past) - 1;
        found = b + at;
        tok0 = (rest - __shfl_sync(kFull, upto - mine, at)) * p.tokens;
      } else {
        rest -= __shfl_sync(kFull, upto, 31);
      }
    }
    if (found < 0) return;
    seq = found;
  }
  if (seq >= live) return;
  Sequence s = sequence(p.batch, seq);
  if (s.n > p.few || tok0 >= s.n) return;
  {  // as a sequence of its own, which ends with its last token
    const int rest = s.n - tok0 - p.tokens;
    s.row0 += tok0;
    s.n = rest > 0 ? p.tokens : s.n - tok0;
    s.kv -= max(rest, 0);
  }
  const int rows = s.n * p.group;
  const int tiles = (rows + 7) / 8;  // 8-row groups that there are
  const int pos0 = s.kv - s.n;  // keys before the first token's own
  const int k0 = split * p.split_keys, k1 = p.splits > 1 ? min(s.kv, k0 + p.split_keys) : s.kv;
  const int64_t row0 = (int64_t)s.row0 * p.hq + kvh * p.group;  // of [token, head] rows
  const int64_t part =
      (((int64_t)split * p.batch.n_seqs + seq) * p.few + tok0) * p.hq + kvh * p.group;
  if (p.splits > 1 && k0 >= k1) {  // no keys: a sum of 0
    for (int r = threadIdx.x; r < rows; r += blockDim.x)
      p.part_ml[part + (int64_t)(r / p.group) * p.hq + r % p.group] = make_float2(-INFINITY, 0.f);
    return;
  }
  unsigned char *ring = dyn + ((1024u - (ptx::smem_u32(dyn) & 1023u)) & 1023u) + warp * F::kRing;
  __syncthreads();

  // this warp's groups of 16 keys: warp, warp + 4, ... of the split's
  const int groups = max(0, ((k1 - k0 + kFewKeys - 1) / kFewKeys - warp + kFewWarps - 1) / kFewWarps);
  const int page = 1 << p.src.page_shift;
  auto key_of = [&](int i) { return k0 + (warp + i * kFewWarps) * kFewKeys; };
  // cache rows of 32 groups at a time, one per lane, the next ones read ahead
  auto cache_rows = [&](int i0) {
    const int i = i0 + lane;
    if (i >= groups) return 0;
    const int at = key_of(i);
    const int pg = __ldg(p.src.tables + s.req * p.src.max_pages + (at >> p.src.page_shift));
    const bool real = pg >= 0 && pg < p.src.n_pages;
    if (!real) raise_error(p.batch.err, TIDE_DEVERR_POSITION);
    // a row past the cache's last reads as zeros
    return ((real ? pg : p.src.n_pages) * p.hkv + (real ? kvh : 0)) * page + (at & (page - 1));
  };
  int now = cache_rows(0), next = cache_rows(32);
  auto request = [&](int i) {
    if (i >= groups) return;
    if ((i & 31) == 0 && i) {
      now = next;
      next = cache_rows(i + 32);
    }
    const int row = __shfl_sync(kFull, now, i & 31);
    const int st = i % kFewStages;
    if (lane == 0) ptx::mbar_expect_tx(&full[warp][st], 2 * F::kSide);
    __syncwarp();
    if (lane < 2 * kHalves)  // K, then V, a column group each
      ptx::tma_load_2d(ring + st * 2 * F::kSide + lane * F::kHalf, lane < kHalves ? &mk : &mv,
                       &full[warp][st], lane % kHalves * 64, row);
    __syncwarp();
  };
  for (int i = 0; i < kFewStages; ++i) request(i);

  // Q^T: columns are rows 8 nt + lane / 4; the statistics of a column are kept
  // by the lanes whose accumulators belong to it, columns 8 nt + 2 (lane % 4)
  // and one further
  uint32_t qb[NT][D / 16][2];
  int sees[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + lane / 4;
    const bool valid = r < rows;
    const T *q = static_cast<const T *>(p.q) + (s.row0 + (valid ? r / p.group : 0)) * p.q_stride +
                 (int64_t)(kvh * p.group + r % p.group) * D + (lane & 3) * 2;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qb[nt][k][e] = valid ? *reinterpret_cast<const uint32_t *>(q + k * 16 + e * 8) : 0u;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = nt * 8 + (lane & 3) * 2 + e;
      sees[nt][e] = pos0 + (c < rows ? c / p.group : s.n - 1) + 1;
    }
  }
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[nt][d][0] = o[nt][d][1] = o[nt][d][2] = o[nt][d][3] = 0.f;
  }
  const float slack = kSlack / p.qs;
  // ldmatrix addresses of this lane within a group: rows of keys, 16-byte chunks
  const int kr = lane & 15, kc = lane >> 4;                             // K: [key][dim]
  const int vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;    // V, transposed
  int i = 0;
  for (; i < groups; ++i) {
    const int st = i % kFewStages;
    if (!__all_sync(kFull, ptx::mbar_wait(&full[warp][st], (i / kFewStages) & 1, &s_abort))) {
      raise_error(p.batch.err, TIDE_DEVERR_TIMEOUT);
      s_abort = 1;
      break;
    }
    const unsigned char *kb = ring + st * 2 * F::kSide, *vb = kb + F::kSide;
    const uint32_t ka = ptx::smem_u32(kb) + kr * 128, va = ptx::smem_u32(vb) + vr * 128;
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int c = k * 2 + kc;
      uint32_t a[4];
      ldmatrix4(a, ka + (c / 8) * F::kHalf + (((c % 8) ^ (kr & 7)) << 4));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (nt < tiles) mma16816<T>(sc[nt], a, qb[nt][k][0], qb[nt][k][1]);
    }
    const int key = key_of(i);
    const bool partial = key + kFewKeys > pos0 + 1;  // some row does not see all of them
    uint32_t pt[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt >= tiles) continue;
      float a[2], x[4];
      bool raise = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // keys lane / 4 and 8 further
        const int lim = sees[nt][e] - key - lane / 4;
        if (partial && lim <= 0) sc[nt][e] = -INFINITY;
        if (partial && lim <= 8) sc[nt][2 + e] = -INFINITY;
        float t = fmaxf(sc[nt][e], sc[nt][2 + e]);
#pragma unroll
        for (int w = 4; w < 32; w *= 2) t = fmaxf(t, __shfl_xor_sync(kFull, t, w));
        const bool up = t > m[nt][e] + slack;  // (the first keys: m is -infinity)
        a[e] = up ? ex2((m[nt][e] - t) * p.qs) : 1.f;
        if (up) m[nt][e] = t;
        raise |= up;
        const float mq = (m[nt][e] == -INFINITY ? 0.f : m[nt][e] * p.qs) - kLift<T>;
        x[e] = ex2(fmaf(sc[nt][e], p.qs, -mq));
        x[2 + e] = ex2(fmaf(sc[nt][2 + e], p.qs, -mq));
        l[nt][e] = fmaf(l[nt][e], a[e], x[e] + x[2 + e]);
      }
      pt[nt][0] = transpose8x8(pack_weights<T>(x[0], x[1]));
      pt[nt][1] = transpose8x8(pack_weights<T>(x[2], x[3]));
      if (__any_sync(kFull, raise)) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          o[nt][d][0] *= a[0];
          o[nt][d][1] *= a[1];
          o[nt][d][2] *= a[0];
          o[nt][d][3] *= a[1];
        }
      }
    }
    // Masked values: a weight of 0 does not silence a NaN.  Past the last key
    // they are dropped; before it, where rows differ, odd ones are taken out,
    // and added to the rows that do see them.
    const int seen = s.kv - key;  // keys of the group that exist
    if (seen < kFewKeys || (partial && s.n > 1)) {
      unsigned char *v = ring + st * 2 * F::kSide + F::kSide;
      constexpr int kRowVecs = 8 * kHalves;
      auto word = [&](int e) {  // word e of the group: keys, then 16-byte vectors
        return reinterpret_cast<uint32_t *>(v + (e / 32 % kHalves) * F::kHalf +
                                            e / (4 * kRowVecs) * 128 + e % 32 * 4);
      };
      bool odd = false;
      for (int e = lane; e < kFewKeys * kRowVecs * 4; e += 32) {
        uint32_t *w = word(e);
        if (e / (4 * kRowVecs) >= seen) *w = 0u;
        else odd |= odd_value<T>(*w) | odd_value<T>(*w >> 16);
      }
      if (__any_sync(kFull, odd)) {
        // rare: key by key, 16-byte chunk and row of the warp's own layout
#pragma unroll 1
        for (int k = 0; k < min(seen, kFewKeys); ++k) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int dim = d * 16 + h * 8 + lane / 4, c = dim / 8;
                const float x = Elem<T>::to_f(*reinterpret_cast<const T *>(
                    v + (c / 8) * F::kHalf + k * 128 + (((c % 8) ^ (k & 7)) << 4) + dim % 8 * 2));
                if (!isfinite(x)) {
                  if (key + k < sees[nt][0]) o[nt][d][h * 2] += x;
                  if (key + k < sees[nt][1]) o[nt][d][h * 2 + 1] += x;
                }
              }
        }
        __syncwarp();
        for (int e = lane; e < kFewKeys * kRowVecs * 4; e += 32) {
          uint32_t *w = word(e);
          if (odd_value<T>(*w)) *w &= 0xFFFF0000u;
          if (odd_value<T>(*w >> 16)) *w &= 0x0000FFFFu;
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const int c = d * 2 + vc;
      uint32_t a[4];
      ldmatrix4_t(a, va + (c / 8) * F::kHalf + (((c % 8) ^ (vr & 7)) << 4));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (nt < tiles) mma16816<T>(o[nt][d], a, pt[nt][0], pt[nt][1]);
    }
    __syncwarp();  // the stage has been read
    ptx::fence_proxy_async();
    request(i + kFewStages);
  }
  if (i < groups && lane == 0) {  // given up: wait for the copies in flight (bounded)
    volatile int none = 0;
    for (int e = i; e < min(groups, i + kFewStages); ++e)
      ptx::mbar_wait(&full[warp][e % kFewStages], (e / kFewStages) & 1, &none);
  }
  __syncwarp();

  // the four warps' outputs meet: this warp's in its own ring, [row][D + 4]
  constexpr int kPitch = D + 4;  // (4: eight lanes of a column write to eight places)
  float *mine = reinterpret_cast<float *>(ring);
  static_assert(kRowsMost * kPitch * 4 <= F::kRing, "a warp's output fits its ring");
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + (lane & 3) * 2 + e;
      float sum = l[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w *= 2) sum += __shfl_xor_sync(kFull, sum, w);
      if (lane < 4) {
        s_m[warp][r] = m[nt][e] * p.qs;
        s_l[warp][r] = sum;
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        mine[r * kPitch + d * 16 + lane / 4] = o[nt][d][e];
        mine[r * kPitch + d * 16 + 8 + lane / 4] = o[nt][d][2 + e];
      }
    }
  __syncthreads();
  const float *all = reinterpret_cast<const float *>(ring - warp * F::kRing);
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
      const float a = exp2f(s_m[w][r] - top);
      const float4 y = *reinterpret_cast<const float4 *>(all + w * (F::kRing / 4) + r * kPitch + d);
      sum = fmaf(a, s_l[w][r], sum);
      x.x = fmaf(a, y.x, x.x);
      x.y = fmaf(a, y.y, x.y);
      x.z = fmaf(a, y.z, x.z);
      x.w = fmaf(a, y.w, x.w);
    }
    const int64_t at = (int64_t)(r / p.group) * p.hq + r % p.group;
    if (p.splits > 1) {
      if (d == 0) p.part_ml[part + at] = make_float2(top, sum);
      *reinterpret_cast<float4 *>(p.part_o + (part + at) * D + d) = x;
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + (row0 + at) * D + d) =
          make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
    }
  }
}

// ------------------------------------------------------------------- joins
// Joins the splits of a row and head: with M = max_s m_s,
//   o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
// `per` warps of the CTA's eight share a row: eight splits each at a time, whose
// loads are all in flight before the first is used (a join is latency), with a
// running maximum; then the warps' results in their order.
// FEW: the rows are [sequence, token below few]; else the packed rows of the
// sequences with more tokens than that.
template <typename T, int D, bool FEW>
__global__ void __launch_bounds__(256)
    join_kernel(const __grid_constant__ RaggedBatch batch, int hq, int few, int splits, int per,
                const float *__restrict__ part_o, const float2 *__restrict__ part_ml, T *out) {
  constexpr int kE = D / 32, kBatch = 8;
  __shared__ float s_m[8], s_l[8], s_o[8][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t step = (int64_t)(FEW ? (int64_t)batch.n_seqs * few : batch.n_tokens) * hq;
  const int64_t at = (int64_t)blockIdx.x * (8 / per) + warp / per;
  const int live = live_sequences(batch);
  int64_t row = -1;
  if (at < step) {
    if (FEW) {
      const int seq = (int)(at / hq / few), tok = (int)(at / hq % few);
      if (seq < live) {
        const Sequence s = sequence(batch, seq);
        if (s.n <= few && tok < s.n) row = s.row0 + tok;
      }
    } else {
      const int seq = sequence_of_row(batch, live, (int)(at / hq));
      if (seq >= 0 && sequence(batch, seq).n > few) row = at / hq;
    }
  }
  // The kernels before waited for what made the batch before they let this one
  // start; what they themselves write comes now.
  ptx::grid_dependency_wait();
  ptx::grid_dependents_launch();
  float m = -INFINITY, l = 0.f, o[kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) o[e] = 0.f;
  if (row >= 0) {
    for (int i0 = warp % per; i0 < splits; i0 += per * kBatch) {
      float2 ml[kBatch];
      float x[kBatch][kE];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = i0 + b * per;
        ml[b] = i < splits ? part_ml[i * step + at] : make_float2(-INFINITY, 0.f);
        const float *src = part_o + (min(i, splits - 1) * step + at) * D + lane * kE;
#pragma unroll
        for (int e = 0; e < kE; ++e) x[b][e] = src[e];  // (not written where the sum is 0)
      }
      float top = m;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) top = ml[b].y != 0.f ? fmaxf(top, ml[b].x) : top;
      const float a = l != 0.f ? exp2f(m - top) : 0.f;
      l *= a;
#pragma unroll
      for (int e = 0; e < kE; ++e) o[e] = l != 0.f ? o[e] * a : 0.f;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (ml[b].y == 0.f) continue;
        const float f = exp2f(ml[b].x - top);
        l = fmaf(f, ml[b].y, l);
#pragma unroll
        for (int e = 0; e < kE; ++e) o[e] = fmaf(f, x[b][e], o[e]);
      }
      m = top;
    }
  }
  if (per > 1) {
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int e = 0; e < kE; ++e) s_o[warp][lane * kE + e] = o[e];
    __syncthreads();
    if (warp % per) return;
    float top = -INFINITY;
    for (int w = warp; w < warp + per; ++w)
      if (s_l[w] != 0.f) top = fmaxf(top, s_m[w]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] = 0.f;
    for (int w = warp; w < warp + per; ++w) {
      if (s_l[w] == 0.f) continue;
      const float f = exp2f(s_m[w] - top);
      l = fmaf(f, s_l[w], l);
#pragma unroll
      for (int e = 0; e < kE; ++e) o[e] = fmaf(f, s_o[w][lane * kE + e], o[e]);
    }
  }
  if (row < 0) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *to = out + (row * hq + at % hq) * D + lane * kE;
#pragma unroll
  for (int e = 0; e < kE; ++e) to[e] = Elem<T>::from_f(o[e] * inv);
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

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> fn{nullptr};
  auto f = fn.load(std::memory_order_acquire);
  if (!f) {
    void *sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) ==
            cudaSuccess && q == cudaDriverEntryPointSuccess)
      f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym);
    fn.store(f, std::memory_order_release);
  }
  return f;
}

// 16-bit rows [d2][d1][d0], s1 and s2 elements apart, in boxes of 64 of a
// row's elements (128 bytes, swizzled; or 32, 64 bytes) by b1 by b2.
bool make_map(CUtensorMap *m, int dtype, const void *base, int rank, int64_t d0, int64_t d1,
              int64_t d2, int64_t s1, int64_t s2, int b1, int b2, int b0 = 64) {
  auto enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2};
  cuuint64_t strides[2] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2};
  cuuint32_t box[3] = {(cuuint32_t)b0, (cuuint32_t)b1, (cuuint32_t)b2};
  cuuint32_t step[3] = {1, 1, 1};
  return enc(m, dtype == TIDE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
             (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE,
             b0 == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The checks that both entry points share; 0 or a status with its message.
int check_heads(int dtype, int64_t hq, int64_t hkv, int64_t d, float scale, int64_t n_tokens,
                int64_t n_seqs) {
  if (dtype != TIDE_DTYPE_BF16 && dtype != TIDE_DTYPE_F16)
    return fail(TIDE_ERR_UNSUPPORTED, "ragged attention: dtype must be bf16 or fp16");
  if (d != 64 && d != 128)
    return fail(TIDE_ERR_UNSUPPORTED, "ragged attention: head_dim must be 64 or 128");
  if (hkv < 1 || hq < 1 || hq % hkv || hq / hkv > tide::ragged::kRows || hq > 65536)
    return fail(TIDE_ERR_INVALID, "ragged attention: bad heads (1 to 128 query heads per KV head)");
  if (!(scale > 0.f) || isinf(scale))
    return fail(TIDE_ERR_INVALID, "ragged attention: scale must be positive and finite");
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2 || n_seqs < 0 || n_seqs > INT32_MAX / 2)
    return fail(TIDE_ERR_INVALID, "ragged attention: bad number of rows or sequences");
  return TIDE_OK;
}

// Units (two tiles, one KV head) that a batch may have at most.
int64_t most_units(int64_t n_tokens, int64_t n_seqs, int64_t hq, int64_t hkv) {
  const int64_t per = 2 * (tide::ragged::kRows / (hq / hkv));
  const int64_t tiles = n_tokens / per + (n_seqs < n_tokens ? n_seqs : n_tokens);
  return tiles * hkv;
}

// How a paged call is cut up.  Sequences of up to `few` tokens (rows that fit
// the few-rows kernel) and longer ones go to a kernel each; a call that cannot
// have the one or the other does not launch it.
struct Plan {
  int nt;                // 8-row groups of a CTA of the few-rows kernel; 0: none
  int few, tokens;
  int64_t pieces;        // of up to `tokens` tokens, at most
  bool tiles;            // whether the tile kernel runs
  int few_splits, split_keys;
  int splits, split_blocks;
  size_t few_bytes, bytes;  // workspace
};

// tiles_only: no few-rows kernel, whatever the sequences.
Plan plan_paged(bool one_token, int64_t n_tokens, int64_t n_seqs, int64_t hq, int64_t hkv, int64_t d,
                int64_t max_kv, bool tiles_only = false) {
  using namespace tide::ragged;
  Plan p{};
  const int64_t group = hq / hkv;
  // Rows of a CTA of the few-rows kernel: 8 for a decode step whose heads fit
  // them, else 16, else 32.
  p.nt = one_token && group <= 8 ? 1 : group <= 16 ? 2 : group <= 32 ? 4 : 0;
  p.tokens = (int)(p.nt * 8 / group);
  // The lengths are on the device; few is what two CTAs take.  mma.sync bounds
  // that kernel from some 16 rows on (16 requests of 1 to 9 tokens and 4 heads
  // each over up to 2100 keys: 54 us there, 41 us as tiles), so with more on
  // average every sequence goes to the tiles; with one sequence its length is
  // known.
  p.few = one_token ? 1 : 2 * p.tokens;
  if (!one_token && (n_tokens * group > n_seqs * 16 || (n_seqs == 1 && n_tokens > p.few))) p.nt = 0;
  if (tiles_only) p.nt = 0;
  if (!p.nt) p.few = 0;
  if (n_tokens < p.few) p.few = (int)n_tokens;
  p.tiles = !p.nt || (!one_token && n_tokens > p.few);
  p.pieces = n_seqs + (p.few > p.tokens ? n_tokens / p.tokens : 0);
  const int64_t rows = n_tokens * hq;
  // Few rows.  Up to a quarter as many units as CTAs that run at once (two an
  // SM): one round of them, with splits of 128 keys at least (3 requests of 9000
  // to 40000 keys, 8 KV heads: 51 us; with up to eight rounds of splits of 512
  // 57; one of 1000: 7.9 and 10.9).  More units: up to eight rounds, since
  // sequences differ in length, and the more pieces, the evener the end (16
  // requests of up to 16000: 98 us in one round, 88 in eight).
  constexpr int64_t kSlots = 2 * 148;
  const int64_t units = p.pieces * hkv;
  const bool one_round = units * 4 <= kSlots;
  const int64_t least = one_round ? 128 : 512;
  int64_t s = !p.nt ? 1 : one_round ? kSlots / units : (8 * kSlots + units - 1) / units;
  if (s > (max_kv + least - 1) / least) s = (max_kv + least - 1) / least;
  if (s < 1 || units >= 4 * 148) s = 1;
  const int64_t keys = (max_kv + s - 1) / s;
  p.split_keys = (int)((keys + 63) / 64 * 64);
  p.few_splits = (int)s;
  p.few_bytes = s > 1 ? (size_t)(s * n_seqs * p.few * hq * (d + 2) * 4 + 15) / 16 * 16 : 0;
  // Tiles: the number of splits whose rounds over the SMs end soonest.  A block
  // of keys takes a unit about 1.8 us, starting and ending it 4 us, and a
  // split's outputs go to HBM and back (8 (d + 2) bytes a row at 6.5 TB/s).
  const int64_t tile_units = most_units(n_tokens, n_seqs, hq, hkv);
  const int64_t blocks = (max_kv + kKeys - 1) / kKeys;
  int64_t t = 1;
  double best = 0;
  for (int64_t i = 1; p.tiles && i <= 32 && (i == 1 || i * 4 <= blocks); ++i) {
    const double rounds = (double)((tile_units * i + 147) / 148);
    const double us = rounds * (1.8 * (double)((blocks + i - 1) / i) + 4.0) +
                      (i > 1 ? 4.0 + 8.0 * (double)(rows * i * (d + 2)) / 6.5e6 : 0.0);
    if (i == 1 || us < best) best = us, t = i;
  }
  p.splits = (int)t;
  p.split_blocks = (int)((blocks + t - 1) / t);
  p.bytes = p.few_bytes + (t > 1 ? (size_t)(t * rows * (d + 2) * 4) : 0);
  return p;
}

template <typename T, int D, bool PAGED>
int launch(tide::ragged::Params &p, int dtype, const void *q, int64_t q_stride, int64_t kv_rows,
           bool behind_few, cudaStream_t s) {
  using namespace tide::ragged;
  CUtensorMap mq, mk, mv, mo;
  const int page = 1 << p.src.page_shift;
  const int box = PAGED && page < kKeys ? page : kKeys;
  bool ok = make_map(&mq, dtype, q, 3, D, p.hq, p.batch.n_tokens, D, q_stride, p.group, p.tokens);
  for (int kv = 0; kv < 2; ++kv) {
    CUtensorMap *m = kv ? &mv : &mk;
    const void *base = kv ? p.src.v : p.src.k;
    ok = ok && (PAGED ? make_map(m, dtype, base, 2, D, kv_rows, 1, D, 0, box, 1)
                      : make_map(m, dtype, base, 3, D, p.hkv, p.batch.n_tokens, D, p.src.row_stride,
                                 1, box));
  }
  p.boxes = 32 % p.group == 0 || p.group % 32 == 0;
  if (p.boxes && p.splits == 1) {
    const int heads = p.group < 32 ? p.group : 32;
    ok = ok && make_map(&mo, dtype, p.out, 3, D, p.hq, p.batch.n_tokens, D, (int64_t)p.hq * D, heads,
                        32 / heads, 32);
  } else {
    mo = mq;  // (not used)
  }
  if (!ok) return fail(TIDE_ERR_CUDA, "ragged attention: cuTensorMapEncodeTiled failed");
  auto kern = tile_attention_kernel<T, D, PAGED>;
  static std::atomic<uint64_t> set{0};  // per device
  cudaError_t e = tide::allow_smem(kern, (int)Shape<D>::kSmem, set);
  if (e != cudaSuccess) return report(e, "ragged attention");
  const int64_t units =
      most_units(p.batch.n_tokens, p.batch.n_seqs, p.hq, p.hkv) * p.splits;
  if (units > INT32_MAX) return fail(TIDE_ERR_INVALID, "ragged attention: too many rows and heads");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)units, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Shape<D>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  p.take_over = units > 148;
  p.behind_few = behind_few;
  return report(cudaLaunchKernelEx(&cfg, kern, p, mq, mk, mv, mo), "ragged attention");
}

template <typename T, int D, int NT>
int launch_few(const tide::ragged::FewParams &p, int dtype, int64_t kv_rows, cudaStream_t s) {
  using namespace tide::ragged;
  CUtensorMap mk, mv;
  if (!make_map(&mk, dtype, p.src.k, 2, D, kv_rows, 1, D, 0, kFewKeys, 1) ||
      !make_map(&mv, dtype, p.src.v, 2, D, kv_rows, 1, D, 0, kFewKeys, 1))
    return fail(TIDE_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed");
  const int64_t ctas = (int64_t)p.pieces * p.hkv * p.splits;
  if (ctas > INT32_MAX) return fail(TIDE_ERR_INVALID, "paged_attention: too many sequences and heads");
  auto kern = few_rows_kernel<T, D, NT>;
  static std::atomic<uint64_t> set{0};  // per device
  cudaError_t e = tide::allow_smem(kern, (int)Few<D>::kSmem, set);
  if (e != cudaSuccess) return report(e, "paged_attention");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3(32 * kFewWarps, 1, 1);
  cfg.dynamicSmemBytes = Few<D>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return report(cudaLaunchKernelEx(&cfg, kern, p, mk, mv), "paged_attention");
}

template <typename T, int D, bool FEW>
int launch_join(const tide::RaggedBatch &b, int hq, int few, int splits, const float *part_o,
                const float2 *part_ml, void *out, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int64_t rows = (int64_t)(FEW ? (int64_t)b.n_seqs * few : b.n_tokens) * hq;
  const int per = splits <= 8 ? 1 : splits <= 16 ? 2 : splits <= 32 ? 4 : 8;
  cfg.gridDim = dim3((unsigned)((rows * per + 7) / 8), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];  // its launch overlaps the tail of the kernel before
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return report(cudaLaunchKernelEx(&cfg, tide::ragged::join_kernel<T, D, FEW>, b, hq, few, splits,
                                   per, part_o, part_ml, static_cast<T *>(out)),
                "paged_attention");
}

// The paged call of one element type and head dimension, as planned.
template <typename T, int D>
int run_paged(const Plan &plan, tide::ragged::Params &p, int dtype, const void *q, int64_t q_stride,
              int64_t kv_rows, unsigned char *ws, cudaStream_t s) {
  const int64_t few_rows = (int64_t)p.batch.n_seqs * plan.few * p.hq;
  const int64_t rows = (int64_t)p.batch.n_tokens * p.hq;
  float *few_o = reinterpret_cast<float *>(ws);
  float2 *few_ml = reinterpret_cast<float2 *>(ws + plan.few_splits * few_rows * D * 4);
  p.few = plan.few;
  if (plan.splits > 1) {
    p.splits = plan.splits;
    p.split_blocks = plan.split_blocks;
    p.part_o = reinterpret_cast<float *>(ws + plan.few_bytes);
    p.part_ml = reinterpret_cast<float2 *>(ws + plan.few_bytes + plan.splits * rows * D * 4);
  }
  int rc;
  if (plan.nt) {
    tide::ragged::FewParams f{p.batch, p.src,  q,     q_stride,  p.out,       few_o,
                              few_ml,  p.hq,   p.hkv, p.group,   plan.few,    plan.tokens,
                              (int)plan.pieces, plan.few_splits, plan.split_keys, p.qs};
    rc = plan.nt == 1   ? launch_few<T, D, 1>(f, dtype, kv_rows, s)
         : plan.nt == 2 ? launch_few<T, D, 2>(f, dtype, kv_rows, s)
                        : launch_few<T, D, 4>(f, dtype, kv_rows, s);
    if (rc) return rc;
  }
  if (plan.tiles && (rc = launch<T, D, true>(p, dtype, q, q_stride, kv_rows, plan.nt != 0, s))) return rc;
  if (plan.nt && plan.few_splits > 1 &&
      (rc = launch_join<T, D, true>(p.batch, p.hq, plan.few, plan.few_splits, few_o, few_ml, p.out, s)))
    return rc;
  if (plan.splits > 1)
    return launch_join<T, D, false>(p.batch, p.hq, plan.few, plan.splits, p.part_o, p.part_ml, p.out, s);
  return TIDE_OK;
}

void set_heads(tide::ragged::Params &p, int64_t hq, int64_t hkv, int64_t d, float scale, void *out) {
  p.out = out;
  p.hq = (int)hq;
  p.hkv = (int)hkv;
  p.group = (int)(hq / hkv);
  p.tokens = tide::ragged::kRows / p.group;
  p.qs = scale * tide::ragged::kLog2e;
  p.splits = 1;
  p.split_blocks = 1 << 24;  // all of them
  p.few = 0;
  p.group_keys = (64 << 20) / (hkv * d * 4);
}

}  // namespace

namespace tide {

size_t paged_tiles_workspace_size(int64_t n_tokens, int64_t n_seqs, int64_t hq, int64_t hkv, int64_t d,
                                  int64_t max_kv) {
  if (n_tokens < 1 || n_seqs < 1 || max_kv < 1) return 0;
  return plan_paged(false, n_tokens, n_seqs, hq, hkv, d, max_kv, true).bytes;
}

int paged_tiles(int dtype, int64_t head_dim, const RaggedBatch &b, const KeySource &src, int few,
                const int32_t *needed, const void *q, int64_t q_stride, void *out, int64_t hq,
                int64_t hkv, float scale, void *workspace, cudaStream_t s) {
  const int64_t d = head_dim, kv_rows = (int64_t)src.n_pages * hkv << src.page_shift;
  Plan plan = plan_paged(false, b.n_tokens, b.n_seqs, hq, hkv, d, b.max_kv, true);
  plan.few = few;
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  ragged::Params p{};
  p.batch = b;
  p.src = src;
  p.needed = needed;
  set_heads(p, hq, hkv, d, scale, out);
  if (dtype == TIDE_DTYPE_BF16)
    return d == 128 ? run_paged<__nv_bfloat16, 128>(plan, p, dtype, q, q_stride, kv_rows, ws, s)
                    : run_paged<__nv_bfloat16, 64>(plan, p, dtype, q, q_stride, kv_rows, ws, s);
  return d == 128 ? run_paged<__half, 128>(plan, p, dtype, q, q_stride, kv_rows, ws, s)
                  : run_paged<__half, 64>(plan, p, dtype, q, q_stride, kv_rows, ws, s);
}

}  // namespace tide

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
  p.zero_keys = zero_keys;
  set_heads(p, n_q_heads, n_kv_heads, head_dim, scale, out);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TIDE_DTYPE_BF16)
    return head_dim == 128
               ? launch<__nv_bfloat16, 128, false>(p, dtype, q, q_row_stride, n_tokens, false, st)
               : launch<__nv_bfloat16, 64, false>(p, dtype, q, q_row_stride, n_tokens, false, st);
  return head_dim == 128 ? launch<__half, 128, false>(p, dtype, q, q_row_stride, n_tokens, false, st)
                         : launch<__half, 64, false>(p, dtype, q, q_row_stride, n_tokens, false, st);
}

extern "C" size_t tide_paged_attention_workspace_size(int64_t n_tokens, int64_t n_seqs,
                                                      int64_t n_q_heads, int64_t n_kv_heads,
                                                      int64_t head_dim, int64_t max_kv_len) {
  if (n_tokens < 1 || n_seqs < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads || max_kv_len < 1 ||
      n_q_heads / n_kv_heads > tide::ragged::kRows)
    return 0;
  // (cu_seqlens or not: the larger need of the two)
  const size_t one = plan_paged(true, n_tokens, n_seqs, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
  const size_t many =
      plan_paged(false, n_tokens, n_seqs, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
  return one > many ? one : many;
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
  const int64_t kv_rows = n_pages * n_kv_heads * page_size;
  cudaStream_t st = (cudaStream_t)stream;
  const Plan plan = plan_paged(!cu_seqlens, n_tokens, n_seqs, n_q_heads, n_kv_heads, head_dim, max_kv_len);
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  tide::ragged::Params p{};
  p.batch = {cu_seqlens, seq_ids, kv_lens, n_seqs_dev, (int)n_seqs, (int)n_requests,
             (int)n_tokens, (int)max_kv_len, error_word};
  p.src = {k_cache, v_cache, 0, block_tables, max_pages, (int)n_pages, shift};
  set_heads(p, n_q_heads, n_kv_heads, head_dim, scale, out);
  if (dtype == TIDE_DTYPE_BF16)
    return head_dim == 128 ? run_paged<__nv_bfloat16, 128>(plan, p, dtype, q, q_row_stride, kv_rows, ws, st)
                           : run_paged<__nv_bfloat16, 64>(plan, p, dtype, q, q_row_stride, kv_rows, ws, st);
  return head_dim == 128 ? run_paged<__half, 128>(plan, p, dtype, q, q_row_stride, kv_rows, ws, st)
                         : run_paged<__half, 64>(plan, p, dtype, q, q_row_stride, kv_rows, ws, st);
}
