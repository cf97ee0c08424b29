// Attention of chunks of new tokens over a paged cache, on the tcgen05 tensor core (formulas:
// paged_attention.cu). Every key byte feeds hundreds of rows, so the two products bound it, and next to
// them the exponentials: two row tiles by 128 positions at head width 128 take 2054 cycles of tensor core
// (2524 with the logits in halves of 64, as here) and 2048 of the SM's 16 exponentials per cycle.
//
// An item is 256 query rows of one key head (rows as in paged.cuh: tokens times the query heads that
// share the key head), as two tiles A and B of 128: while the tensor core multiplies for one, the other's
// logits become weights. One CTA per SM, 16 warps (the last two idle):
//   warps 0-3, 4-7   tiles A, B: a thread owns a query row. It loads the row's Q into shared memory (128-byte
//                    swizzle, K-major), then per 64 positions reads its logits from its TMEM lane and writes
//                    P = 2^(s - m) in 16 bits over the first 32 columns of them, the A operand of the second
//                    product. The reference m moves a few times per row only (Reference in
//                    paged_attention.cuh), since O in TMEM is rescaled with it. At the end it reads its row of O.
//   warps 8-11       K and V tiles of 128 positions into a ring of stages; rows that are not there read as
//                    zero, and a bit per row says so. Pages of 8, 16, 32, .. positions: warp 8 issues one TMA
//                    box per page and 64 elements, a lane each (a page that is not there is a coordinate past
//                    the pool, which TMA fills with zeros), and warps 9-11 search values in positions that
//                    not every row sees for infinities and NaN. Other page sizes: all four warps gather rows
//                    with 16-byte cp.async (3300 cycles a tile, 2355 us where the boxes take 1402).
//   warps 12, 13     issue S = Q K^T (M = 128, N = 64) and O += P V (P from TMEM, V MN-major as it lies in
//                    the cache) for a tile each, in the order PV(i) S(i + 2): the two halves of a tile's 128
//                    logit columns are two buffers, and the tensor core runs a thread's instructions in issue
//                    order, so a commit of S(i + 2) also says that PV(i) is done.
// TMEM: S/P of A 0-127, of B 128-255, O of A 256-383, of B 384-511.
//
// Measured (2000 tokens over 40009 positions, 32 query and 8 key heads of 128, bf16, page 64): 1480 to 1560 us
// on several cards, 820 to 865 TFLOP/s, 0.52 of the measured bf16 rate; the tensor pipe is active 49% of the
// cycles, the exponentials' as much. What bounds it is the row warps' latency (two per scheduler: logits read, exponentials, weights stored and
// handed over, about 2000 cycles per half against 1145 for the same instructions free of waits). Tried
// without gain, on a card that took 1380: whole 128-column logits (1402), a polynomial for 1 to 4 of 8 exponential pairs (1350-1440),
// tile B kept out of A's exponentials (1460), logits read again instead of kept for the second try (1400).
//
// Waits are bounded: one that runs out sets the error word, every role leaves its loop, the rows of the
// piece are written as NaN, and the CTA ends once its copies and products in flight have.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "paged_attention.cuh"

namespace sb {
namespace k {
namespace {

constexpr int kChunkRows = 256;
constexpr int kChunkKeys = 128;
constexpr int kChunkThreads = 512;
constexpr int kLoadWarp = 8, kMmaWarp = 12;
template <int DP> constexpr int kRing = DP == 128 ? 5 : 8;          // stages of one K or V tile
template <int DP> constexpr uint32_t kTileBytes = 128u * DP * 2;
template <int DP> constexpr int kChunkSmem = int((2 + kRing<DP>) * kTileBytes<DP>) + 1024;
constexpr int kLag = 2;          // stages that a loader keeps in flight
constexpr int kBook = 8;         // entries of the rings of row bits and poison marks

__device__ unsigned chunk_error;   // bits of the waits that ran out since it was last read

constexpr uint32_t kSleepNs = 20000;
constexpr WaitLimit kEndWait = {kWaitTimeoutNs, kSleepNs};   // of what was issued, whatever the other waits' limit

// mbar_wait whose attempts may sleep in hardware until the phase ends (up to 20 us each): the waiting
// warps of the other roles share the row warps' issue slots.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort_flag, WaitLimit limit,
                                           unsigned int code) {
  uint64_t t0 = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(limit.sleep_ns)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > limit.ns) {
      *abort_flag = 1;
      atomicOr(&chunk_error, code);
      return false;
    }
  }
}

// byte offset of 16-byte piece `c` of row `r` in a tile of 128-byte-swizzled slabs of 64 elements
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return uint32_t(c >> 3) * 16384u + uint32_t(r) * 128u + (uint32_t((c & 7) ^ (r & 7)) << 4);
}

template <typename T> constexpr uint32_t kIdescType = 0;
template <> constexpr uint32_t kIdescType<__nv_bfloat16> = (1u << 7) | (1u << 10);
template <typename T> constexpr uint32_t idesc16(int M, int N) {
  return (1u << 4) | kIdescType<T> | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

__device__ __forceinline__ float max3(float x, float y, float z) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
  return d;
}

// v = -infinity where `seen` is 0. (Volatile, so that it stays inside its branch: as selects, the 64 of a
// row's half would be executed for tiles that need none, twice as many instructions as the rest.)
__device__ __forceinline__ void hide(uint32_t& v, uint32_t seen) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\tselp.b32 %0, %0, 0xff800000, p;\n\t}" : "+r"(v) : "r"(seen));
}

// One CTA's walk over its pieces; every role steps through the same ones.
struct Walk {
  int group, window;
  Share sh;
  int64_t u;
  int b, h, i, at;
  SeqWork s;
  // the piece
  int tile_a, tile_b;   // key tiles of the pair
  bool whole, head;     // the item in one piece; the item begins here
  int tiles, first_tile, last_tile;
  int slot;
  int ta0, tb0, ta1, tb1;   // key tiles of A and B in the piece
  int kbeg, kend;
  int64_t all_lo, all_hi;   // positions that every row of the pair sees

  __device__ __forceinline__ void start(const PagedView& c, int g, int win, const Share& share) {
    group = g, window = win, sh = share;
    u = sh.u0, b = sh.b, h = sh.h, i = sh.i, at = sh.tile;
    s = seq_work(c, b, group);
    piece();
  }
  __device__ __forceinline__ void piece() {
    const RowTile<kChunkRows, kChunkKeys> rt(s, i, group, window);
    tiles = rt.tiles;
    const int take = int(min(int64_t(tiles - at), sh.u1 - u));
    tile_a = rt.tile0 + at;
    tile_b = tile_a + take;
    whole = at == 0 && take == tiles;
    head = at == 0;
    kbeg = rt.kbeg, kend = rt.kend;
    all_hi = rt.pos_lo;
    all_lo = window > 0 ? rt.pos_hi - window + 1 : 0;
    slot = 2 * int(blockIdx.x) + (u == sh.u0 ? 0 : 1);
    half(0, ta0, tb0);
    half(1, ta1, tb1);
  }
  __device__ __forceinline__ void half(int x, int& lo, int& hi) const {
    lo = hi = 0;
    if ((2 * i + x) * 128 >= s.rows) return;
    const RowTile<128, kChunkKeys> part(s, 2 * i + x, group, window);
    if (part.kbeg >= part.kend) return;
    lo = max(tile_a, part.tile0);
    hi = min(tile_b, part.tile0 + part.tiles);
    if (lo >= hi) lo = hi = 0;
  }
  __device__ __forceinline__ bool next(const PagedView& c) {
    u += tile_b - tile_a;
    at = 0;
    if (u >= sh.u1) return false;
    if ((++i) * kChunkRows >= s.rows) {
      i = 0;
      if (++h == c.kv_heads) {
        h = 0;
        do {
          if (++b >= c.batch) return false;
          s = seq_work(c, b, group);
        } while (s.rows == 0);
      }
    }
    piece();
    return true;
  }
  __device__ __forceinline__ int ta(int x) const { return x ? ta1 : ta0; }
  __device__ __forceinline__ int tb(int x) const { return x ? tb1 : tb0; }
  // whether some row does not see some position of the tile
  __device__ __forceinline__ bool mixed(int tile) const {
    const int64_t key0 = int64_t(tile) * kChunkKeys;
    return key0 + kChunkKeys - 1 > all_hi || key0 < all_lo;
  }
};

// Takes the infinities and NaNs out of one 16-byte piece of a value tile: a product with a weight of zero
// would carry them to rows that do not see the position. The rows that see them add them at the end. An
// exponent of all ones carries into the sign bit when one is added to it, which finds them two at a time.
template <typename T>
__device__ __forceinline__ bool clean_piece(uint8_t* tile_at, int r, int piece) {
  constexpr uint32_t kExps = Mma<T>::kExp * 0x00010001u, kOnes = (0x8000u - Mma<T>::kExp) * 0x00010001u;
  uint4* at = reinterpret_cast<uint4*>(tile_at + tile_off(r, piece));
  const uint4 v = *at;
  const uint32_t hit = ((v.x & kExps) + kOnes) | ((v.y & kExps) + kOnes) | ((v.z & kExps) + kOnes) | ((v.w & kExps) + kOnes);
  if (!(hit & 0x80008000u)) return false;
  uint16_t* e = reinterpret_cast<uint16_t*>(at);
#pragma unroll
  for (int q = 0; q < 8; ++q)
    if ((e[q] & Mma<T>::kExp) == Mma<T>::kExp) e[q] = 0;
  return true;
}

// Boxes of a whole page, or of 128 of its positions, by 64 elements; rows 0: the cache is gathered.
struct PagedMaps {
  CUtensorMap k, v;
};

template <typename T, int DP, bool kTma>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_chunk_kernel(const PagedArgs a, const __grid_constant__ PagedMaps maps) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int kNst = kRing<DP>;
  constexpr uint32_t kTile = kTileBytes<DP>;
  constexpr int kPieces = DP / 8;
  __shared__ uint64_t full[kNst], empty[kNst], clean[kNst], q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], ended[2];
  __shared__ uint32_t there[kBook][4];      // which of a key tile's 128 positions are there
  __shared__ int poison[kBook];             // number of the last piece that met non-finite values in mixed positions
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  __shared__ Walk row_walk[8];              // of the row warps: their registers hold logits
  volatile int* abort_flag = &abort_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;                       // Q of A, Q of B
  uint8_t* ring = smem + 2 * kTile;
  const PagedView& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = c.head_dim, G = a.group;
  pdl_launch_dependents();

  if (tid == 0) {
    for (int x = 0; x < kNst; ++x) {
      mbar_init(&full[x], kTma ? 1u : 4u);
      mbar_init(&clean[x], 3u);
      mbar_init(&empty[x], kTma ? 5u : 2u);   // both tiles' products, and the three cleaning warps
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 4u);
      mbar_init(&ended[x], 1u);
      for (int y = 0; y < 2; ++y) {
        mbar_init(&s_full[x][y], 1u);
        mbar_init(&p_full[x][y], 4u);
        mbar_init(&pv_done[x][y], 1u);
      }
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < kBook) poison[tid] = 0;
  const Share sh = find_share<kChunkRows, kChunkKeys, kChunkThreads>(c, G, a.window, a.least, blockIdx.x, a.ctas,
                                                                     reinterpret_cast<int64_t*>(smem));
  if (tid < 2) a.notes[2 * blockIdx.x + tid] = PartialNote{0, 0, 0, 0};
  if (sh.u0 >= sh.u1) return;
  if (warp == kMmaWarp) tmem_alloc(&tmem_holder, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;

  // 512 threads start with 128 registers each; 2 x 128 x 168 and 2 x 128 x 88 are the same 65536.
  if (warp < kLoadWarp) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");

  if (warp < kLoadWarp) {
    // ---- rows: Q, softmax, output ----
    Walk& w = row_walk[warp];
    {
      Walk first;
      first.start(c, G, a.window, sh);
      if (lane == 0) w = first;
      __syncwarp();
    }
    auto advance = [&] {
      Walk now = w;
      __syncwarp();
      const bool more = now.next(c);
      if (lane == 0) w = now;
      __syncwarp();
      return more;
    };
    const int x = warp >> 2;                              // tile A or B
    const int r = tid & 127;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t ts_x = tmem + lanes + uint32_t(x * 128), to = tmem + lanes + 256u + uint32_t(x * 128);
    uint8_t* q_at = sq + x * kTile;
    int step = 0;                                         // halves of key tiles before the current piece (even)
    int number = 0, book = 0;                             // pieces, key tiles before the current piece
    do {
      ++number;
      const int row = w.i * kChunkRows + x * 128 + r;
      const bool live = row < w.s.rows;
      const int tok = live ? row / G : 0;
      const int head = w.h * G + (live ? row - tok * G : 0);
      const int64_t pos = w.s.ctx - w.s.n + tok;
      // positions that the row sees: [see_lo, see_hi]
      const int see_hi = live ? int(min(pos, int64_t(w.kend) - 1)) : -1;
      const int see_lo = a.window > 0 ? int(max(pos - a.window + 1, int64_t(0))) : 0;
      const bool busy = w.ta(x) < w.tb(x);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      if (busy) {
        const T* qp = static_cast<const T*>(a.q.p) + (w.s.first + tok) * a.q.ts + int64_t(head) * a.q.hs;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (live && p * 8 < D) v = *reinterpret_cast<const uint4*>(qp + p * 8);
          *reinterpret_cast<uint4*>(q_at + tile_off(r, p)) = v;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[x]);
        const int ta = w.ta(x), steps = 2 * (w.tb(x) - ta), book_a = book + ta - w.tile_a;
        for (int i = 0; i < steps; ++i) {
          const int buf = i & 1;
          ok = __all_sync(~0u, wait_phase(&s_full[x][buf], uint32_t((step + i) >> 1) & 1u, abort_flag, a.wait, 1u));
          if (!ok) break;
          tc_fence_after();
          const int key0 = (ta + (i >> 1)) * kChunkKeys + buf * 64;
          const uint32_t ts = ts_x + uint32_t(buf * 64);
          const uint32_t* bits = there[(book_a + (i >> 1)) % kBook] + buf * 2;
          uint32_t v[64];
          tmem_ld32_async(ts, v);
          tmem_ld32_async(ts + 32, v + 32);
          // every row of the warp sees every position of the half
          const bool plain = __all_sync(~0u, (bits[0] & bits[1]) == ~0u && (!live || (see_hi >= key0 + 63 && see_lo <= key0)));
          tmem_ld_wait(v);
          tmem_ld_wait(v + 32);
          if (!plain) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int lo = see_lo - key0 - g * 32, hi = see_hi - key0 - g * 32;   // in [0, 31] once clamped
              uint32_t mask = hi < 0 ? 0u : hi >= 31 ? ~0u : (2u << hi) - 1u;
              mask &= lo <= 0 ? ~0u : lo > 31 ? 0u : ~((1u << lo) - 1u);
              mask &= bits[g];
#pragma unroll
              for (int j = 0; j < 32; ++j) hide(v[g * 32 + j], mask & (1u << j));
            }
          }
          // The weights are taken against the reference of the steps before, side by side with the maximum; where
          // that is too far from it (a row's first step, and a few after it), once more against a new one.
          float2 sum0, sum1;
          for (bool moved = false;; moved = true) {
            const float base = m == -INFINITY ? 0.f : m - Reference<T>::kLift;
            const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), base2 = make_float2(-base, -base);
            float tops[2] = {-INFINITY, -INFINITY};
            sum0 = sum1 = make_float2(0.f, 0.f);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t pk[16];
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float2 e = make_float2(__uint_as_float(v[g * 32 + j]), __uint_as_float(v[g * 32 + j + 1]));
                tops[(j >> 1) & 1] = max3(tops[(j >> 1) & 1], e.x, e.y);
                e = __ffma2_rn(e, scale2, base2);
                e.x = exp2_approx(e.x);
                e.y = exp2_approx(e.y);
                if (j & 2) sum1 = __fadd2_rn(sum1, e);
                else sum0 = __fadd2_rn(sum0, e);
                pk[j >> 1] = Mma<T>::pack(e.x, e.y);
              }
              tmem_st16(ts + g * 16, pk);
            }
            const float top = fmaxf(tops[0], tops[1]) * a.scale_log2;
            const bool rise = rises<T>(top - m), fall = falls<T>(top - m) && l < kMostSum;
            if (moved || !__any_sync(~0u, rise || fall)) break;
            const float now = rise ? top : fall ? fmaxf(top + kBack, m - kDeepest) : m;
            const float f = rise || fall ? exp2_approx(m - now) : 1.f;   // 0 on a row's first
            m = now;
            l *= f;
            if (i > 0) {
              ok = __all_sync(~0u, wait_phase(&pv_done[x][buf ^ 1], uint32_t((step + i - 1) >> 1) & 1u, abort_flag, a.wait, 2u));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int g = 0; g < DP / 16; ++g) {
                uint32_t o[16];
                tmem_ld16(to + g * 16, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                tmem_st16(to + g * 16, o);
              }
              tmem_st_wait();
            }
          }
          if (!ok) break;
          l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x][buf]);
        }
        step += steps;
        if (ok) ok = __all_sync(~0u, wait_phase(&pv_done[x][1], uint32_t((step - 1) >> 1) & 1u, abort_flag, a.wait, 2u));
        tc_fence_after();
      }
      // ---- the row's result ----
      // The mark may be a later piece's by now: nothing holds the other roles back while this tile has no keys in the
      // pieces after this one. A later one only means that this piece is searched too.
      const bool marked = poison[number % kBook] >= number;
      const float bad = ok ? 0.f : __int_as_float(0x7fc00000);
      const float inv = (l == 0.f ? 0.f : 1.f / l) + bad;
#pragma unroll 1
      for (int g = 0; g < DP / 32; ++g) {
        uint32_t v[32];
        __syncwarp();
        if (busy && ok) {
          tmem_ld32(to + g * 32, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(bad);
        }
        if (!live) continue;
        if (marked) {
          const int32_t* table = c.table + int64_t(w.b) * c.table_stride;
          for (int key = max(w.tile_a * kChunkKeys, w.kbeg); key < min(w.tile_b * kChunkKeys, w.kend); ++key) {
            if (key >= w.all_lo && key <= w.all_hi) {
              key = int(min(w.all_hi, int64_t(w.kend)));   // on to the ones that not all rows see
              continue;
            }
            if (key > see_hi || key < see_lo) continue;
            const int page = table[key / c.page_size];
            if (page < 0 || page >= c.pages) continue;
            const uint16_t* vp = reinterpret_cast<const uint16_t*>(static_cast<const T*>(c.v) + page * c.vp +
                                                                   (key % c.page_size) * c.vt + int64_t(w.h) * c.vh);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (g * 32 + j < D) {
                const uint16_t bits = vp[g * 32 + j];
                if ((bits & Mma<T>::kExp) == Mma<T>::kExp) v[j] = __float_as_uint(__uint_as_float(v[j]) + Mma<T>::widen(bits));
              }
          }
        }
        if (w.whole) {
          T* dst = static_cast<T*>(a.out.p) + (w.s.first + tok) * a.out.ts + int64_t(head) * a.out.hs + g * 32;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            if (g * 32 + p * 8 >= D) break;
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[e] = Mma<T>::pack(__uint_as_float(v[8 * p + 2 * e]) * inv, __uint_as_float(v[8 * p + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + p * 8) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        } else {
          float4* dst = reinterpret_cast<float4*>(a.o + int64_t(w.slot) * (kChunkRows * DP)) + g * 8 * kChunkRows + x * 128 + r;
#pragma unroll
          for (int p = 0; p < 8; ++p)
            dst[p * kChunkRows] = make_float4(__uint_as_float(v[4 * p]), __uint_as_float(v[4 * p + 1]), __uint_as_float(v[4 * p + 2]),
                                              __uint_as_float(v[4 * p + 3]));
        }
      }
      if (!w.whole && live) a.ml[int64_t(w.slot) * kChunkRows + x * 128 + r] = make_float2(m, l + bad);
      if (!w.whole && w.head && tid == 0)
        a.notes[w.slot] = PartialNote{w.b, w.h, w.i, int((w.u + w.tiles - 1) / w.sh.per) - int(blockIdx.x)};
      tc_fence_before();   // these reads of O come before the next piece's products
      book += w.tile_b - w.tile_a;
      if (__any_sync(~0u, *abort_flag)) break;
    } while (advance());
    tmem_st_wait();   // weights of a step that a wait broke off
  } else if (kTma && warp == kLoadWarp) {
    // ---- keys and values: TMA ----
    Walk w;
    w.start(c, G, a.window, sh);
    const int rows = min(c.page_size, kChunkKeys);         // of a box
    const int per_tile = kChunkKeys / rows, boxes = per_tile * (DP / 64);
    const int part = lane % per_tile, slab = lane / per_tile;
    int stage = 0, book = 0;
    bool ok = true;
    do {
      const int32_t* table = c.table + int64_t(w.b) * c.table_stride;
      const int n = w.tile_b - w.tile_a;
      int next = 0, row = 0, page = 0, page_was = 0;       // `pages` for one that is not there
      auto look_up = [&](int tile) {
        const int key = tile * kChunkKeys + part * rows;
        next = int(c.pages);
        if (tile < w.tile_b && key < w.kend && key + rows > w.kbeg) {
          const int p = table[key / c.page_size];
          if (p >= 0 && p < c.pages) next = p;
        }
      };
      look_up(w.tile_a);
      for (int e = 0; e < 2 * n; ++e) {
        const bool value = e == 2 * n - 1 || (e > 0 && (e & 1) == 0);
        const int tile = w.tile_a + (e == 0 ? 0 : value ? (e == 2 * n - 1 ? n - 1 : e / 2 - 1) : (e + 1) / 2);
        const int slot = stage % kNst;
        if (!value) {
          page_was = page;
          page = next;
        }
        const int from = value && e != 2 * n - 1 ? page_was : page;   // the last value's rows are the latest looked up
        row = rows == c.page_size ? 0 : tile * kChunkKeys % c.page_size;
        if (stage >= kNst)
          ok = __all_sync(~0u, wait_phase(&empty[slot], uint32_t((stage / kNst - 1) & 1), abort_flag, a.wait, 4u));
        if (!ok) break;
        if (!value) {
          const uint32_t held = __ballot_sync(~0u, from < c.pages);   // bit p: box p's page is there
          if (lane < 4) {
            uint32_t bits = 0;
            if (rows >= 32) bits = (held >> (lane * 32 / rows)) & 1u ? ~0u : 0u;
            else
              for (int p = 0; p < 32 / rows; ++p)
                if ((held >> (lane * (32 / rows) + p)) & 1u) bits |= ((1u << rows) - 1u) << (p * rows);
            there[(book + tile - w.tile_a) % kBook][lane] = bits;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_expect_tx(&full[slot], kTile);
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(smem_u32(ring + slot * kTile) + uint32_t(slab) * 16384u + uint32_t(part * rows) * 128u, value ? &maps.v : &maps.k,
                      slab * 64, row, w.h, from, &full[slot]);
        if (!value) look_up(tile + 1);
        ++stage;
      }
      book += n;
      if (!ok || __any_sync(~0u, *abort_flag)) break;
    } while (w.next(c));
    // the copies in flight land before this CTA's shared memory is given up
    volatile int not_aborted = 0;
    for (int st = max(0, stage - kNst); st < stage; ++st)
      wait_phase(&full[st % kNst], uint32_t((st / kNst) & 1), &not_aborted, kEndWait, 64u);
  } else if (kTma && warp < kMmaWarp) {
    // ---- non-finite values that not every row sees ----
    Walk w;
    w.start(c, G, a.window, sh);
    const int cw = warp - kLoadWarp - 1;
    int stage = 0, number = 0;
    bool ok = true;
    do {
      ++number;
      const int n = w.tile_b - w.tile_a;
      for (int e = 0; e < 2 * n; ++e, ++stage) {   // every stage: a wait may not skip a phase
        const int slot = stage % kNst;
        ok = __all_sync(~0u, wait_phase(&full[slot], uint32_t((stage / kNst) & 1), abort_flag, a.wait, 128u));
        if (!ok) break;
        const bool value = e == 2 * n - 1 || (e > 0 && (e & 1) == 0);
        const int tile = w.tile_a + (e == 2 * n - 1 ? n - 1 : e / 2 - 1);
        if (value && w.mixed(tile)) {
          // rows [0, below) and [above, 128) hold positions that not every row sees
          const int64_t key0 = int64_t(tile) * kChunkKeys;
          int below = int(clamp64(w.all_lo - key0, 0, kChunkKeys)), above = int(clamp64(w.all_hi + 1 - key0, 0, kChunkKeys));
          if (below > above) below = above = 0;
          const int gap = above - below;
          bool bad = false;
#pragma unroll 1   // (unrolled by four, windowed prompts take 177 us instead of 141: more code beside the row warps')
          for (int p = cw * 32 + lane; p < (kChunkKeys - gap) * kPieces; p += 96) {
            const int r = p / kPieces;
            bad |= clean_piece<T>(ring + slot * kTile, r < below ? r : r + gap, p % kPieces);
          }
          if (bad) poison[number % kBook] = number;
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&clean[slot]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[slot]);
      }
      if (!ok || __any_sync(~0u, *abort_flag)) break;
    } while (w.next(c));
  } else if (!kTma && warp >= kLoadWarp && warp < kMmaWarp) {
    // ---- keys and values: gathered ----
    Walk w;
    w.start(c, G, a.window, sh);
    const int lw = warp - kLoadWarp;
    int stage = 0, number = 0, book = 0;   // stages used, pieces, key tiles before the current piece
    bool ok = true;
    // values of the stages in flight that have positions not every row sees: what to clean when they land
    int clean_tile[kLag + 1], clean_slot[kLag + 1];
#pragma unroll
    for (int j = 0; j <= kLag; ++j) clean_tile[j] = -1, clean_slot[j] = 0;
    int arrived = 0;                       // stages handed over
    int page = -1, in_page = 0, page_was = -1, in_page_was = 0;
    auto hand_over = [&](int tile, int number_of, const Walk& wk) {
      // cleans the pieces that this thread copied, then passes the stage on
      const int slot = arrived % kNst;
      if (tile >= 0) {
        bool bad = false;
#pragma unroll 1
        for (int j = 0; j < kPieces; ++j)
        {
          const int r = lw * 32 + j * (32 / kPieces) + lane / kPieces;
          const int64_t key = int64_t(tile) * kChunkKeys + r;
          if (key > wk.all_hi || key < wk.all_lo) bad |= clean_piece<T>(ring + slot * kTile, r, lane % kPieces);
        }
        if (bad) poison[number_of % kBook] = number_of;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[slot]);
      ++arrived;
    };
    do {
      ++number;
      const int32_t* table = c.table + int64_t(w.b) * c.table_stride;
      const T* kc = static_cast<const T*>(c.k) + int64_t(w.h) * c.kh;
      const T* vc = static_cast<const T*>(c.v) + int64_t(w.h) * c.vh;
      // per piece: K(a), then K(j + 1), V(j) for each tile j
      const int n = w.tile_b - w.tile_a;
      int next_page = -1, next_row = 0;       // of the key tile to load next
      auto look_up = [&](int tile) {
        const int key = tile * kChunkKeys + lw * 32 + lane;
        next_page = -1;
        if (tile < w.tile_b && key >= w.kbeg && key < w.kend) {
          const int page_no = key / c.page_size;
          next_row = key - page_no * c.page_size;
          next_page = table[page_no];
          if (next_page < 0 || next_page >= c.pages) next_page = -1;
        }
      };
      look_up(w.tile_a);
      for (int e = 0; e < 2 * n && ok; ++e) {
        const bool value = e == 2 * n - 1 || (e > 0 && (e & 1) == 0);
        const int tile = w.tile_a + (e == 0 ? 0 : value ? (e == 2 * n - 1 ? n - 1 : e / 2 - 1) : (e + 1) / 2);
        const int slot = stage % kNst;
        if (!value) {
          page_was = page, in_page_was = in_page;
          page = next_page, in_page = next_row;
        }
        const bool last_value = e == 2 * n - 1;    // its rows are the latest looked up
        const int pg = value && !last_value ? page_was : page, ip = value && !last_value ? in_page_was : in_page;
        if (stage >= kNst)
          ok = __all_sync(~0u, wait_phase(&empty[slot], uint32_t((stage / kNst - 1) & 1), abort_flag, a.wait, 4u));
        if (!ok) break;
        if (!value) {
          const uint32_t bits = __ballot_sync(~0u, pg >= 0);
          if (lane == 0) there[(book + tile - w.tile_a) % kBook][lw] = bits;
        }
        const uint32_t dst = smem_u32(ring + slot * kTile);
        const int piece = lane % kPieces;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
          const int rr = j * (32 / kPieces) + lane / kPieces;
          const int p = __shfl_sync(~0u, pg, rr), ri = __shfl_sync(~0u, ip, rr);
          const bool live = p >= 0 && piece * 8 < D;
          const T* src = value ? vc + p * c.vp + ri * c.vt : kc + p * c.kp + ri * c.kt;
          cp_async_16(dst + tile_off(lw * 32 + rr, piece), live ? src + piece * 8 : static_cast<const T*>(c.k), live ? 16u : 0u);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (!value) look_up(tile + 1);
        const bool mixed = value && w.mixed(tile);
#pragma unroll
        for (int j = kLag; j > 0; --j) clean_tile[j] = clean_tile[j - 1];
        clean_tile[0] = mixed ? tile : -1;
        ++stage;
        if (stage - arrived > kLag) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
          hand_over(clean_tile[kLag], number, w);
        }
      }
      // The stages still in flight are handed over here: their cleaning needs this piece's bounds.
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      while (ok && arrived < stage) hand_over(stage - arrived == 2 ? clean_tile[1] : clean_tile[0], number, w);
      book += n;
      if (!ok || __any_sync(~0u, *abort_flag)) break;
    } while (w.next(c));
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    // ---- products: a warp per row tile ----
    const int x = warp - kMmaWarp;
    if (x < 2 && lane == 0) {
      constexpr uint32_t id_s = idesc16<T>(128, 64), id_o = idesc16<T>(128, DP) | kMnMajorB;
      const uint32_t ts = tmem + uint32_t(x * 128), to = tmem + 256u + uint32_t(x * 128);
    Walk w;
    w.start(c, G, a.window, sh);
      const uint64_t qd = sw128_desc(smem_u32(sq + x * kTile));
      int stage = 0, step = 0;
      uint32_t q_phase = 0, clean_phase = 0;
      bool ok = true;
      auto wait_stage = [&](int st) {
        return wait_phase(&full[st % kNst], uint32_t((st / kNst) & 1), abort_flag, a.wait, 8u);
      };
      auto logits = [&](int st, int half) {   // 64 positions
        const uint64_t kd = sw128_desc(smem_u32(ring + (st % kNst) * kTile) + uint32_t(half) * 8192u);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t at = uint64_t((kk >> 2) * 1024 + (kk & 3) * 2);   // a slab of 64 elements is 16 KB
          umma_bf16(ts + uint32_t(half * 64), qd + at, kd + at, id_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[x][half]);
      };
      do {
        const int n = w.tile_b - w.tile_a, ta = w.ta(x), tb = w.tb(x);
        // stages of this piece: K(a) is 0; K(j) is 2j - 1; V(j) is 2j + 2, but the last V is 2n - 1
        auto k_stage = [&](int j) { return stage + (j == 0 ? 0 : 2 * j - 1); };
        auto v_stage = [&](int j) { return stage + (j == n - 1 ? 2 * n - 1 : 2 * j + 2); };
        if (ta < tb) {
          ok = wait_phase(&q_full[x], q_phase, abort_flag, a.wait, 16u);
          q_phase ^= 1u;
        }
        ok = ok && wait_stage(k_stage(0));
        if (!ok) break;
        tc_fence_after();
        if (w.tile_a >= ta && w.tile_a < tb) {
          logits(k_stage(0), 0);
          logits(k_stage(0), 1);
        }
        umma_commit(&empty[k_stage(0) % kNst]);
        for (int j = 0; j < n && ok; ++j) {
          const int tile = w.tile_a + j;
          const bool on = tile >= ta && tile < tb, on_next = j + 1 < n && tile + 1 >= ta && tile + 1 < tb;
          ok = wait_stage(v_stage(j));
          if (kTma && ok && w.mixed(tile)) {
            const int slot = v_stage(j) % kNst;
            ok = wait_phase(&clean[slot], (clean_phase >> slot) & 1u, abort_flag, a.wait, 256u);
            clean_phase ^= 1u << slot;
          }
          if (!ok) break;
          const uint64_t vd = sw128_mn_desc(smem_u32(ring + (v_stage(j) % kNst) * kTile), 16384u);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (on) {
              ok = ok && wait_phase(&p_full[x][half], uint32_t(step >> 1) & 1u, abort_flag, a.wait, 32u);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)   // 16 positions: two 8-row groups of 1024 B
                umma_f16_ts(to, ts + uint32_t(half * 64 + kk * 8), vd + uint64_t(half * 512 + kk * 128), id_o,
                            tile > ta || half > 0 || kk > 0 ? 1u : 0u);
              umma_commit(&pv_done[x][half]);
              ++step;
            }
            if (half == 1) umma_commit(&empty[v_stage(j) % kNst]);
            if (half == 0 && j + 1 < n) {
              ok = wait_stage(k_stage(j + 1));
              if (!ok) break;
              tc_fence_after();
            }
            if (on_next) logits(k_stage(j + 1), half);
          }
          if (!ok) break;
          if (j + 1 < n) umma_commit(&empty[k_stage(j + 1) % kNst]);
        }
        stage += 2 * n;
      } while (ok && w.next(c));
      // The products in flight, and the arrivals of the last releases, come before this CTA's memory is given up.
      volatile int not_aborted = 0;
      umma_commit(&ended[x]);
      wait_phase(&ended[x], 0u, &not_aborted, kEndWait, 512u);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  // Items that begin here and end elsewhere are not joined if some of this CTA's warps left before their last piece.
  if (tid < 2 && abort_word) a.notes[2 * blockIdx.x + tid].more = 0;
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of each split item in the order of their positions: a thread per row and 4 elements.
template <typename T, int DP>
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const PagedArgs a) {
  pdl_wait();
  const PartialNote n0 = a.notes[2 * blockIdx.x], n1 = a.notes[2 * blockIdx.x + 1];
  const bool second = n1.more > 0;
  if (!second && n0.more <= 0) return;
  const PartialNote n = second ? n1 : n0;
  const SeqWork s = seq_work(a.c, n.b, a.group);
  const int r = threadIdx.x, row = n.i * kChunkRows + r;
  if (row >= s.rows) return;
  const int64_t first = int64_t(2 * blockIdx.x + (second ? 1 : 0)), next = 2 * (int64_t(blockIdx.x) + 1);
  float top = -INFINITY;
  for (int p = 0; p <= n.more; ++p) top = fmaxf(top, a.ml[(p == 0 ? first : next + 2 * (p - 1)) * kChunkRows + r].x);
  const float base = top == -INFINITY ? 0.f : top;
  const int tok = row / a.group;
  T* to = static_cast<T*>(a.out.p) + (s.first + tok) * a.out.ts + int64_t(n.h * a.group + row - tok * a.group) * a.out.hs;
  float sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  const int d4 = blockIdx.y;
  for (int p = 0; p <= n.more; ++p) {
    const int64_t slot = p == 0 ? first : next + 2 * (p - 1);
    const float2 ml = a.ml[slot * kChunkRows + r];
    const float f = exp2_approx(ml.x - base);
    const float4 o = reinterpret_cast<const float4*>(a.o + slot * (kChunkRows * DP))[d4 * kChunkRows + r];
    sum += f * ml.y;
    v.x += f * o.x;
    v.y += f * o.y;
    v.z += f * o.z;
    v.w += f * o.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (d4 * 4 < a.c.head_dim)
    *reinterpret_cast<uint2*>(to + d4 * 4) = make_uint2(Mma<T>::pack(v.x * inv, v.y * inv), Mma<T>::pack(v.z * inv, v.w * inv));
}

// The cache as (element, position in page, head, page); false where TMA cannot describe it.
bool encode_pages(CUtensorMap* tm, const void* base, const PagedView& c, int64_t page, int64_t token, int64_t head, bool bf16) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p) : nullptr;
  }();
  const int rows = std::min(c.page_size, kChunkKeys);
  if (!fn || rows < 8 || kChunkKeys % rows != 0 || c.page_size % rows != 0 || c.pages < 1) return false;
  const int64_t stride[3] = {token, head, page};
  const cuuint64_t dims[4] = {cuuint64_t(c.head_dim), cuuint64_t(c.page_size), cuuint64_t(c.kv_heads), cuuint64_t(c.pages)};
  cuuint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] == 1) bytes[i] = 16;   // never stepped along
    else if (stride[i] <= 0 || stride[i] >= (int64_t(1) << 39)) return false;
    else bytes[i] = cuuint64_t(stride[i]) * 2;
  }
  const cuuint32_t box[4] = {64, cuuint32_t(rows), 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, bytes, box,
            step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, bool kTma>
cudaError_t launch_chunk(const PagedArgs& a, const PagedMaps& maps, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(paged_chunk_kernel<T, DP, kTma>, kChunkSmem<DP>, done);
  if (e != cudaSuccess) return e;
  paged_chunk_kernel<T, DP, kTma><<<a.ctas, kChunkThreads, kChunkSmem<DP>, s>>>(a, maps);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_dependent(paged_chunk_join_kernel<T, DP>, dim3(unsigned(a.ctas), DP / 4), 256, a, s);
}

template <typename T, int DP>
cudaError_t launch_chunk(const PagedArgs& a, cudaStream_t s) {
  PagedMaps maps = {};
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const PagedView& c = a.c;
  const bool tma = encode_pages(&maps.k, c.k, c, c.kp, c.kt, c.kh, bf16) && encode_pages(&maps.v, c.v, c, c.vp, c.vt, c.vh, bf16);
  return tma ? launch_chunk<T, DP, true>(a, maps, s) : launch_chunk<T, DP, false>(a, maps, s);
}

__global__ void forget_errors_kernel(unsigned bits) { atomicAnd(&chunk_error, ~bits); }

// SHOROKOO_B200_WAIT_NS: a limit by which a test sees waits run out
WaitLimit wait_limit() {
  static const uint64_t ns = [] {
    const char* e = std::getenv("SHOROKOO_B200_WAIT_NS");
    const unsigned long long v = e ? std::strtoull(e, nullptr, 10) : 0;
    return v > 0 && v < kWaitTimeoutNs ? uint64_t(v) : kWaitTimeoutNs;
  }();
  return {ns, uint32_t(std::min<uint64_t>(ns, kSleepNs))};
}

}  // namespace

// Clears no more than it reports: a wait on another stream may run out in between.
cudaError_t paged_wait_errors(unsigned* bits, cudaStream_t s) {
  void* at = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&at, chunk_error);
  if (e == cudaSuccess) e = cudaMemcpyAsync(bits, at, sizeof(*bits), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess || *bits == 0) return e;
  forget_errors_kernel<<<1, 1, 0, s>>>(*bits);
  e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e;
}

// More than 32 query rows per sequence and key head, on average over the batch: the host knows no more, so that a
// step of single tokens and a prompt's chunk goes to one kernel as a whole. 16 sequences, all alike, over 4000 positions (32 query, 8 key
// heads of 128): at 12 rows the 16-row kernel takes 62 us and this one 101, at 24 and 32 both 101 (it reads the
// cache once per 16 rows), at 48 rows 152 and 102.
bool paged_chunk_wanted(const PagedView& c) {
  return c.batch > 0 && c.tokens * (c.q_heads / c.kv_heads) > 32 * int64_t(c.batch);
}

PagedSpace paged_chunk_space(const PagedView& c, int sms) {
  PagedSpace z;
  z.dp = c.head_dim <= 64 ? 64 : 128;
  z.ctas = sms;
  z.notes = up256(size_t(z.ctas) * 2 * sizeof(PartialNote));
  z.ml = up256(size_t(z.ctas) * 2 * kChunkRows * sizeof(float2));
  z.o = up256(size_t(z.ctas) * 2 * kChunkRows * z.dp * sizeof(float));
  return z;
}

cudaError_t paged_chunk(const PagedView& c, int elem, HeadsView q, HeadsView out, float scale, int window, void* ws, int sms,
                        cudaStream_t s) {
  const PagedSpace z = paged_chunk_space(c, sms);
  PagedArgs a;
  a.c = c, a.q = q, a.out = out;
  a.group = c.q_heads / c.kv_heads, a.window = window, a.ctas = z.ctas;
  // Key tiles of a CTA, at least: 300 tokens over 8000 positions 81.5 us with 1 to 8; 100 over 2000 29.2, 29.3, 32.5
  // and 41.9 with 1, 2, 4 and 8; a prompt of 500 38.9, 38.9, 52.0 and 79.8. (Short prompts
  // would be faster with 2.)
  a.least = 4;
  a.wait = wait_limit();
  a.scale_log2 = scale * 1.4426950408889634f;
  uint8_t* p = static_cast<uint8_t*>(ws);
  a.notes = reinterpret_cast<PartialNote*>(p);
  a.ml = reinterpret_cast<float2*>(p + z.notes);
  a.o = reinterpret_cast<float*>(p + z.notes + z.ml);
  if (elem == 10) return z.dp == 64 ? launch_chunk<__half, 64>(a, s) : launch_chunk<__half, 128>(a, s);
  return z.dp == 64 ? launch_chunk<__nv_bfloat16, 64>(a, s) : launch_chunk<__nv_bfloat16, 128>(a, s);
}

}  // namespace k
}  // namespace sb
