// Device helpers of the kernels over a paged cache: a sequence's rows and context, read with every
// bound checked, so that no content of the index arrays leads outside the buffers.
#pragma once

#include "decoder.h"

namespace sb {
namespace k {
namespace {

// Rows [first, end) of the step's packed tensors belong to the sequence; its context ends at ctx.
struct SeqRows {
  int64_t first, end, ctx;
};

__host__ __device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

__host__ __device__ __forceinline__ SeqRows seq_rows(const PagedView& c, int b) {
  SeqRows s;
  s.first = clamp64(c.starts[b], 0, c.tokens);
  s.end = clamp64(c.starts[b + 1], s.first, c.tokens);
  s.ctx = c.ctx[b] > 0 ? c.ctx[b] : 0;
  return s;
}

// The last sequence that starts at or before `token` (whole warp; 32 candidates per step).
__device__ __forceinline__ int find_sequence(const PagedView& c, int64_t token) {
  int lo = 0, range = c.batch;   // the answer is in [lo, lo + range)
  const int lane = threadIdx.x & 31;
  while (range > 1) {
    const int step = (range + 31) / 32;
    const int at = lo + lane * step;
    const bool le = lane * step < range && c.starts[at] <= token;
    const unsigned hits = __ballot_sync(~0u, le);
    const int last = hits ? 31 - __clz(hits) : 0;
    lo += last * step;
    range = min(step, range - last * step);
  }
  return lo;
}

// ---- work of the attention kernels ----
// An item is (sequence b, key head h, row tile i): up to `kRows` query rows that read one key head's
// keys, row r being token r / group, head h * group + r % group of the sequence. Its work is its tiles
// of `kKeys` positions, those that any of its rows sees (one, if none does). All items' tiles, in the
// order (b, h, i, tile), are cut into equal consecutive ranges, one per CTA, whatever the sequences'
// lengths are; an item that a cut splits leaves partial results that are joined afterwards.

// A sequence as the attention kernels see it: rows, and the positions its rows may see.
struct SeqWork {
  int64_t first;       // row of its first token
  int64_t ctx;         // its context as given
  int n;               // tokens
  int rows;            // n * group
  int kmax;            // positions that its table can hold, at most ctx
};

__host__ __device__ __forceinline__ SeqWork seq_work(const PagedView& c, int b, int group) {
  const SeqRows r = seq_rows(c, b);
  SeqWork s;
  s.first = r.first;
  s.ctx = r.ctx;
  s.n = int(r.end - r.first);
  s.rows = s.n * group;
  const int64_t cap = int64_t(c.max_pages) * c.page_size;
  s.kmax = int(r.ctx < cap ? r.ctx : cap);
  return s;
}

// Row tile i of a sequence: its rows, and positions [kbeg, kend) that one or more of them see; the
// ones in [lo_all, hi_all] are seen by all of them.
template <int kRows, int kKeys>
struct RowTile {
  int r0, rows;
  int kbeg, kend;
  int64_t pos_lo, pos_hi;   // positions of its first and last token
  int tile0, tiles;         // key tiles from kbeg / kKeys

  __host__ __device__ __forceinline__ RowTile(const SeqWork& s, int i, int group, int window) {
    r0 = i * kRows;
    rows = s.rows - r0 < kRows ? s.rows - r0 : kRows;
    const int64_t pos0 = s.ctx - s.n;
    pos_lo = pos0 + r0 / group;
    pos_hi = pos0 + (r0 + rows - 1) / group;
    kend = int(clamp64(pos_hi + 1, 0, s.kmax));
    kbeg = window > 0 ? int(clamp64(pos_lo - window + 1, 0, kend)) : 0;
    tile0 = kbeg / kKeys;
    const int last = (kend + kKeys - 1) / kKeys;
    tiles = kbeg < kend ? last - tile0 : 1;
  }
};

template <int kRows, int kKeys>
__device__ __forceinline__ int64_t seq_tiles(const SeqWork& s, int group, int window) {
  int64_t sum = 0;
  for (int i = 0; i * kRows < s.rows; ++i) sum += RowTile<kRows, kKeys>(s, i, group, window).tiles;
  return sum;
}

// The share of a CTA: [u0, u1) of all tiles, beginning `tile` tiles into item (b, h, i).
struct Share {
  int64_t u0, u1, per;
  int b, h, i, tile;
};

// Every CTA works its share out by itself (whole block; the result is the same in all threads): the
// sequences' tiles are counted by a thread each, or by a warp each where they have many row tiles,
// and summed; then the sequence, head and row tile that hold its first tile are looked up. `count` is
// kCounted words of shared memory that are free until then.
constexpr int kCounted = 512;   // sequences whose counts are kept between the two steps

template <int kRows, int kKeys, int kThreads>
__device__ __forceinline__ Share find_share(const PagedView& c, int group, int window, int least, int cta, int ctas, int64_t* count) {
  __shared__ int64_t warp_sum[kThreads / 32];
  __shared__ int64_t found_rem;
  __shared__ Share found;
  using Tile = RowTile<kRows, kKeys>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool kept = c.batch <= kCounted;
  int64_t own = 0;
  if (kept && c.tokens * group > int64_t(2 * kRows) * c.batch) {
    for (int b = warp; b < c.batch; b += kThreads / 32) {
      const SeqWork s = seq_work(c, b, group);
      int64_t n = 0;
      for (int i = lane; i * kRows < s.rows; i += 32) n += Tile(s, i, group, window).tiles;
#pragma unroll
      for (int d = 16; d; d >>= 1) n += __shfl_xor_sync(~0u, n, d);
      n *= c.kv_heads;
      if (lane == 0) {
        count[b] = n;
        own += n;
      }
    }
  } else {
    for (int b = tid; b < c.batch; b += kThreads) {
      const int64_t n = seq_tiles<kRows, kKeys>(seq_work(c, b, group), group, window) * c.kv_heads;
      if (kept) count[b] = n;
      own += n;
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) own += __shfl_xor_sync(~0u, own, d);
  if (lane == 0) warp_sum[warp] = own;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += warp_sum[w];
  Share s;
  s.per = (total + ctas - 1) / ctas;
  if (s.per < least) s.per = least;
  s.u0 = s.per * cta;
  s.u1 = s.u0 + s.per < total ? s.u0 + s.per : total;
  if (s.u0 >= s.u1) return s;
  int64_t before = 0;   // tiles of the sequences before this round of kThreads
  for (int b0 = 0; b0 < c.batch; b0 += kThreads) {
    const int b = b0 + tid;
    int64_t mine = 0;
    if (b < c.batch)
      mine = kept ? count[b] : seq_tiles<kRows, kKeys>(seq_work(c, b, group), group, window) * c.kv_heads;
    int64_t upto = mine;   // inclusive sum over the block's threads
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += v;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) upto += warp_sum[w];
      all += warp_sum[w];
    }
    upto += before;
    if (s.u0 < upto && s.u0 >= upto - mine) {
      const int64_t per_head = mine / c.kv_heads, rem = s.u0 - (upto - mine);
      s.b = b;
      s.h = int(rem / per_head);
      found = s;
      found_rem = rem - s.h * per_head;
    }
    before += all;
    if (s.u0 < before) break;   // uniform
  }
  __syncthreads();
  if (warp == 0) {   // 32 row tiles at a time
    const SeqWork sw = seq_work(c, found.b, group);
    int64_t rem = found_rem;
    for (int i0 = 0; i0 * kRows < sw.rows; i0 += 32) {
      const int i = i0 + lane;
      const int64_t t = i * kRows < sw.rows ? Tile(sw, i, group, window).tiles : 0;
      int64_t upto = t;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t v = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += v;
      }
      const bool here = rem < upto && rem >= upto - t;
      if (here) {
        found.i = i;
        found.tile = int(rem - (upto - t));
      }
      if (__any_sync(~0u, here)) break;
      rem -= __shfl_sync(~0u, upto, 31);
    }
  }
  __syncthreads();
  return found;
}

}  // namespace
}  // namespace k
}  // namespace sb
