// Attention of new tokens over a paged cache: o = softmax(scale q k^T) v, one pass over the keys with
// a running maximum and sum per query row (base 2: scale * log2(e) is folded into the exponent):
//   m' = max(m, max_j s_j),  l' = l 2^(m - m') + sum_j 2^(s_j - m'),  o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j
// Two partial results over disjoint keys join the same way, which is what splits a context over CTAs.
// m, l and o are fp32; the weights are rounded to the operands' 16-bit type for the second product, by at most
// 2^-8 (bf16) or 2^-11 (fp16) of each weight, in either direction, as the result itself is: the tensor core takes no
// wider operand with 16-bit values. (Reference in paged_attention.cuh: how fp16's range is kept from losing weights.)
//
// paged_rows_kernel: 16 query rows per item, for decode steps (the q_heads / kv_heads query heads that
// share a key head, times a few tokens). Each byte of the cache feeds 2 x rows operations: reading keys
// and values bounds it. The products run on mma m16n8k16: at 16 rows the tensor core's legacy path has
// several times the rate that the memory can feed, and needs no operand staging beyond shared memory.
// Each of a CTA's 4 warps takes 16 of a tile's 64 positions, with its own ring of stages (cp.async, no
// barrier between warps) and its own m, l, o, joined in shared memory at the item's end.
//
// Measured (bf16, 32 query and 8 key heads of 128, page 16): 48 sequences of up to 8000 positions 168 us replayed
// from a graph, 5.5 TB/s, 0.85 of the measured HBM rate (170 to 180 called from Python); with the arithmetic taken
// out of the first version's 171 us 150, so the loads' pattern is sound and what is left is the warps' own latency
// per stage. Three CTAs per SM with two stages each: 173 us; one CTA with six stages: 282 us.
#include <algorithm>

#include "paged_attention.cuh"

namespace sb {
namespace k {
namespace {

constexpr int kRowsTile = 16;
constexpr int kKeysTile = 64;
constexpr int kRowsThreads = 128;
template <int DP> constexpr int kStages = DP == 128 ? 3 : 4;
template <int DP> constexpr int kRowsSmem = 4 * kStages<DP> * 2 * 16 * DP * 2;

template <typename T, int DP>
__global__ void __launch_bounds__(kRowsThreads, 2) paged_rows_kernel(const PagedArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t held[4][kStages<DP>];   // which of a stage's 16 positions are there
  __shared__ float2 warp_ml[4][kRowsTile];
  __shared__ int poisoned;
  using Tile = RowTile<kRowsTile, kKeysTile>;
  constexpr int kNst = kStages<DP>;
  constexpr int kChunks = DP / 8;                    // 16-byte pieces of a row
  constexpr uint32_t kPart = 16 * DP * 2, kStage = 2 * kPart;
  const PagedView& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int D = c.head_dim, G = a.group;
  pdl_launch_dependents();

  Share sh = find_share<kRowsTile, kKeysTile, kRowsThreads>(c, G, a.window, a.least, blockIdx.x, a.ctas,
                                                              reinterpret_cast<int64_t*>(smem));
  if (tid < 2) a.notes[2 * blockIdx.x + tid] = PartialNote{0, 0, 0, 0};
  if (sh.u0 >= sh.u1) return;
  __syncthreads();

  uint8_t* ring = smem + warp * (kNst * kStage);
  const uint32_t ring_at = smem_u32(ring);
  int64_t u = sh.u0;
  int b = sh.b, h = sh.h, i = sh.i, at = sh.tile;
  SeqWork s = seq_work(c, b, G);
  while (u < sh.u1) {
    const Tile rt(s, i, G, a.window);
    const int take = int(min(int64_t(rt.tiles - at), sh.u1 - u));
    const int tile_a = rt.tile0 + at, tile_b = tile_a + take;
    const bool whole = at == 0 && take == rt.tiles;
    __syncthreads();   // the shared memory of the piece before is free
    if (tid == 0) poisoned = 0;
    __syncthreads();

    // ---- keys and values through the warp's ring ----
    const int32_t* table = c.table + int64_t(b) * c.table_stride;
    const T* kc = static_cast<const T*>(c.k) + int64_t(h) * c.kh;
    const T* vc = static_cast<const T*>(c.v) + int64_t(h) * c.vh;
    int next_page = -1, next_row = 0;   // lanes 0-15: of the next tile to load
    auto look_up = [&](int tile) {
      next_page = -1;
      const int key = tile * kKeysTile + warp * 16 + (lane & 15);
      if (tile < tile_b && key >= rt.kbeg && key < rt.kend) {
        const int page_no = key / c.page_size;
        next_row = key - page_no * c.page_size;
        next_page = table[page_no];
        if (next_page < 0 || next_page >= c.pages) next_page = -1;
      }
    };
    auto load = [&](int tile, int stage) {
      const uint32_t mask = __ballot_sync(~0u, next_page >= 0) & 0xffffu;
      if (lane == 0) held[warp][stage] = mask;
      const uint32_t dst = ring_at + stage * kStage;
      const int chunk = lane % kChunks;
#pragma unroll
      for (int r0 = 0; r0 < 16; r0 += 32 / kChunks) {
        const int r = r0 + lane / kChunks;
        const int page = __shfl_sync(~0u, next_page, r), row = __shfl_sync(~0u, next_row, r);
        const bool live = page >= 0 && chunk * 8 < D;
        const uint32_t to = dst + r * (DP * 2) + ((chunk ^ (r & 7)) << 4);
        const T* kp = live ? kc + page * c.kp + row * c.kt + chunk * 8 : static_cast<const T*>(c.k);
        const T* vp = live ? vc + page * c.vp + row * c.vt + chunk * 8 : static_cast<const T*>(c.v);
        cp_async_16(to, kp, live ? 16u : 0u);
        cp_async_16(to + kPart, vp, live ? 16u : 0u);
      }
    };
    look_up(tile_a);
#pragma unroll
    for (int p = 0; p < kNst - 1; ++p) {
      if (tile_a + p < tile_b) load(tile_a + p, p);
      asm volatile("cp.async.commit_group;" ::: "memory");
      look_up(tile_a + p + 1);
    }

    // ---- this item's queries as operands of S = Q K^T ----
    uint32_t qf[DP / 16][4];
    int64_t pos[2];   // positions of rows g and g + 8
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = g + e * 8;
      const bool live = r < rt.rows;
      const int row = rt.r0 + (live ? r : 0), tok = row / G;
      pos[e] = s.ctx - s.n + tok;
      const T* qp = static_cast<const T*>(a.q.p) + (s.first + tok) * a.q.ts + int64_t(h * G + row - tok * G) * a.q.hs;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = ks * 16 + 2 * t;
        qf[ks][e] = live && d < D ? *reinterpret_cast<const uint32_t*>(qp + d) : 0u;
        qf[ks][e + 2] = live && d + 8 < D ? *reinterpret_cast<const uint32_t*>(qp + d + 8) : 0u;
      }
    }
    // positions that some row does not see: above `all_hi` or below `all_lo`
    const int64_t all_hi = rt.pos_lo, all_lo = a.window > 0 ? rt.pos_hi - a.window + 1 : 0;

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    int stage = 0, to_stage = kNst - 1;
    for (int tile = tile_a; tile < tile_b; ++tile) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kNst - 2) : "memory");
      __syncwarp();   // all lanes' pieces are there, and all lanes are done with the stage refilled next
      if (tile + kNst - 1 < tile_b) load(tile + kNst - 1, to_stage);
      asm volatile("cp.async.commit_group;" ::: "memory");
      look_up(tile + kNst);
      const int key0 = tile * kKeysTile + warp * 16;
      const uint32_t mask = held[warp][stage];
      const uint32_t kat = ring_at + stage * kStage, vat = kat + kPart;
      const bool mixed = key0 + 15 > all_hi || key0 < all_lo;   // not every row sees every position

      float sc[2][4], odd[2][4];   // two sums each: half as long a chain of dependent products
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[e][0] = sc[e][1] = sc[e][2] = sc[e][3] = 0.f;
        odd[e][0] = odd[e][1] = odd[e][2] = odd[e][3] = 0.f;
      }
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        uint32_t kf[4];
        const int r = (lane & 7) + ((lane & 16) >> 1), chunk = 2 * ks + ((lane & 8) >> 3);
        ldmatrix4(kf, kat + r * (DP * 2) + ((chunk ^ (r & 7)) << 4));
        Mma<T>::run(ks & 1 ? odd[0] : sc[0], qf[ks], kf[0], kf[1]);
        Mma<T>::run(ks & 1 ? odd[1] : sc[1], qf[ks], kf[2], kf[3]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[e][j] = (sc[e][j] + odd[e][j]) * a.scale_log2;
      if (mask != 0xffffu || mixed) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int kk = e * 8 + 2 * t + (j & 1);
            const int64_t key = key0 + kk, p = pos[j >> 1];
            const bool seen = ((mask >> kk) & 1u) && key <= p && (a.window == 0 || key > p - a.window);
            if (!seen) sc[e][j] = -INFINITY;
          }
      }
      if (mixed) {
        // A value that only some rows see must not reach the others through a product with zero: its
        // infinities and NaNs are taken out here and added to the rows that see it at the end.
        bool bad = false;
        for (int p = lane; p < 16 * kChunks; p += 32) {
          const int r = p / kChunks, chunk = p - r * kChunks;
          const int64_t key = key0 + r;
          if (key <= all_hi && key >= all_lo) continue;
          uint16_t* e = reinterpret_cast<uint16_t*>(ring + stage * kStage + kPart + r * (DP * 2) + ((chunk ^ (r & 7)) << 4));
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((e[j] & Mma<T>::kExp) == Mma<T>::kExp) {
              e[j] = 0;
              bad = true;
            }
        }
        if (bad) poisoned = 1;
        __syncwarp();
      }
      // The rows' references m move only when one has to, so that most steps need no exchange between lanes and
      // leave o alone.
      float top[2];
      bool moves = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {   // rows g, g + 8
        top[e] = fmaxf(fmaxf(sc[0][2 * e], sc[0][2 * e + 1]), fmaxf(sc[1][2 * e], sc[1][2 * e + 1]));
        moves |= rises<T>(top[e] - m[e]) || falls<T>(top[e] - m[e]);
      }
      if (__any_sync(~0u, moves)) {
        float grow[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 2));
          float now = fmaxf(m[e], top[e]);
          if (Reference<T>::kFalls) {
            float sum = l[e];
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            if (falls<T>(top[e] - m[e]) && sum < kMostSum) now = fmaxf(top[e] + kBack, m[e] - kDeepest);
          }
          grow[e] = exp2_approx(m[e] - (now == -INFINITY ? 0.f : now));
          m[e] = now;
          l[e] *= grow[e];
        }
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
          o[j][0] *= grow[0];
          o[j][1] *= grow[0];
          o[j][2] *= grow[1];
          o[j][3] *= grow[1];
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[e] == -INFINITY ? 0.f : m[e] - Reference<T>::kLift;   // a row that has seen nothing yet
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = exp2_approx(sc[j >> 1][2 * e + (j & 1)] - base);
        l[e] += (p[0] + p[1]) + (p[2] + p[3]);
        pf[e] = Mma<T>::pack(p[0], p[1]);
        pf[e + 2] = Mma<T>::pack(p[2], p[3]);
      }
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        uint32_t vf[4];
        const int r = lane & 15, chunk = 2 * j + (lane >> 4);
        ldmatrix4_trans(vf, vat + r * (DP * 2) + ((chunk ^ (r & 7)) << 4));
        Mma<T>::run(o[2 * j], pf, vf[0], vf[1]);
        Mma<T>::run(o[2 * j + 1], pf, vf[2], vf[3]);
      }
      stage = stage + 1 == kNst ? 0 : stage + 1;
      to_stage = to_stage + 1 == kNst ? 0 : to_stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(~0u, l[e], 1);
      l[e] += __shfl_xor_sync(~0u, l[e], 2);
    }

    // ---- join the four warps ----
    if (t == 0) {
      warp_ml[warp][g] = make_float2(m[0], l[0]);
      warp_ml[warp][g + 8] = make_float2(m[1], l[1]);
    }
    __syncthreads();   // every warp is done with its ring
    float* part = reinterpret_cast<float*>(smem);   // [4][16][DP + 8]
    constexpr int kPitch = DP + 8;
    static_assert(4 * 16 * kPitch * 4 <= kRowsSmem<DP>, "the rings hold the warps' results");
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) {
      float* p0 = part + (warp * 16 + g) * kPitch + j * 8 + 2 * t;
      *reinterpret_cast<float2*>(p0) = make_float2(o[j][0], o[j][1]);
      *reinterpret_cast<float2*>(p0 + 8 * kPitch) = make_float2(o[j][2], o[j][3]);
    }
    __syncthreads();
    const int slot = 2 * blockIdx.x + (u == sh.u0 ? 0 : 1);
    for (int x = tid; x < rt.rows * (DP / 4); x += kRowsThreads) {
      const int r = x / (DP / 4), d = (x - r * (DP / 4)) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, warp_ml[w][r].x);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = exp2_approx(warp_ml[w][r].x - base);
        const float4 p = *reinterpret_cast<const float4*>(part + (w * 16 + r) * kPitch + d);
        sum += f * warp_ml[w][r].y;
        v.x += f * p.x;
        v.y += f * p.y;
        v.z += f * p.z;
        v.w += f * p.w;
      }
      const int row = rt.r0 + r, tok = row / G;
      if (poisoned && d < D) {
        const int64_t p = s.ctx - s.n + tok;
        float* e = &v.x;
        for (int key = max(tile_a * kKeysTile, rt.kbeg); key < min(tile_b * kKeysTile, rt.kend); ++key) {
          if (key >= all_lo && key <= all_hi) {
            key = int(min(all_hi, int64_t(rt.kend)));   // on to the ones that not all see
            continue;
          }
          if (key > p || (a.window > 0 && key <= p - a.window)) continue;
          const int page = table[key / c.page_size];
          if (page < 0 || page >= c.pages) continue;
          const T* vp = vc + page * c.vp + (key % c.page_size) * c.vt + d;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint16_t bits = reinterpret_cast<const uint16_t*>(vp)[j];
            if ((bits & Mma<T>::kExp) == Mma<T>::kExp) e[j] += Mma<T>::widen(bits);
          }
        }
      }
      if (whole) {
        if (d < D) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          T* to = static_cast<T*>(a.out.p) + (s.first + tok) * a.out.ts + int64_t(h * G + row - tok * G) * a.out.hs + d;
          *reinterpret_cast<uint2*>(to) = make_uint2(Mma<T>::pack(v.x * inv, v.y * inv), Mma<T>::pack(v.z * inv, v.w * inv));
        }
      } else {
        *reinterpret_cast<float4*>(a.o + (int64_t(slot) * kRowsTile + r) * DP + d) = v;
        if (d == 0) a.ml[int64_t(slot) * kRowsTile + r] = make_float2(top, sum);
      }
    }
    if (!whole && at == 0 && tid == 0)
      a.notes[slot] = PartialNote{b, h, i, int((u + rt.tiles - 1) / sh.per) - int(blockIdx.x)};

    u += take;
    at = 0;
    if ((++i) * kRowsTile >= s.rows) {
      i = 0;
      if (++h == c.kv_heads) {
        h = 0;
        do {
          if (++b >= c.batch) return;
          s = seq_work(c, b, G);
        } while (s.rows == 0);
      }
    }
  }
}

// Joins the pieces of each split item in the order of their positions: a warp per row.
template <typename T, int DP, int kRows>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a) {
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PartialNote n0 = a.notes[2 * blockIdx.x], n1 = a.notes[2 * blockIdx.x + 1];
  const bool second = n1.more > 0;
  if (!second && n0.more <= 0) return;
  const PartialNote n = second ? n1 : n0;
  const SeqWork s = seq_work(a.c, n.b, a.group);
  const int r = blockIdx.y * 4 + warp, row = n.i * kRows + r;
  if (r >= kRows || row >= s.rows) return;
  const int64_t first = int64_t(2 * blockIdx.x + (second ? 1 : 0)), next = 2 * (int64_t(blockIdx.x) + 1);
  auto slot = [&](int p) { return (p == 0 ? first : next + 2 * (p - 1)) * kRows + r; };
  const int pieces = n.more + 1;
  float top = -INFINITY;
  for (int p = lane; p < pieces; p += 32) top = fmaxf(top, a.ml[slot(p)].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  const float base = top == -INFINITY ? 0.f : top;
  constexpr int kPer = DP / 32;
  float v[kPer] = {}, sum = 0.f;
  for (int p0 = 0; p0 < pieces; p0 += 32) {
    float f = 0.f, l = 0.f;   // of piece p0 + lane
    if (p0 + lane < pieces) {
      const float2 ml = a.ml[slot(p0 + lane)];
      f = exp2_approx(ml.x - base);
      l = f * ml.y;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
    sum += l;
    const int count = min(32, pieces - p0);
#pragma unroll 8
    for (int p = 0; p < count; ++p) {
      const float w = __shfl_sync(~0u, f, p);
      const float* o = a.o + slot(p0 + p) * DP + lane * kPer;
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] += w * o[j];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int tok = row / a.group, d = lane * kPer;
  T* to = static_cast<T*>(a.out.p) + (s.first + tok) * a.out.ts + int64_t(n.h * a.group + row - tok * a.group) * a.out.hs + d;
  if (d < a.c.head_dim) {
#pragma unroll
    for (int j = 0; j < kPer; j += 2) *reinterpret_cast<uint32_t*>(to + j) = Mma<T>::pack(v[j] * inv, v[j + 1] * inv);
  }
}

PagedSpace space(const PagedView& c, int sms) {
  PagedSpace z;
  z.dp = c.head_dim <= 64 ? 64 : 128;
  z.ctas = 2 * sms;
  z.notes = up256(size_t(z.ctas) * 2 * sizeof(PartialNote));
  z.ml = up256(size_t(z.ctas) * 2 * kRowsTile * sizeof(float2));
  z.o = up256(size_t(z.ctas) * 2 * kRowsTile * z.dp * sizeof(float));
  return z;
}

template <typename T, int DP>
cudaError_t launch_rows(PagedArgs a, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(paged_rows_kernel<T, DP>, kRowsSmem<DP>, done);
  if (e != cudaSuccess) return e;
  paged_rows_kernel<T, DP><<<a.ctas, kRowsThreads, kRowsSmem<DP>, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_dependent(paged_join_kernel<T, DP, kRowsTile>, dim3(unsigned(a.ctas), kRowsTile / 4), 128, a, s);
}

}  // namespace

size_t paged_attention_workspace(const PagedView& c, int sms) {
  const PagedSpace z = paged_chunk_wanted(c) ? paged_chunk_space(c, sms) : space(c, sms);
  return z.notes + z.ml + z.o;
}

cudaError_t paged_attention(const PagedView& c, int elem, HeadsView q, HeadsView out, float scale, int window, void* ws, int sms,
                            cudaStream_t s) {
  if (paged_chunk_wanted(c)) return paged_chunk(c, elem, q, out, scale, window, ws, sms, s);
  const PagedSpace z = space(c, sms);
  PagedArgs a;
  a.c = c, a.q = q, a.out = out;
  a.group = c.q_heads / c.kv_heads, a.window = window, a.ctas = z.ctas;
  // Key tiles of a CTA, at least: one sequence over 1500 positions 18.8, 15.4, 15.3 and 19.7 us with 1, 2, 4 and 8;
  // over 256 positions 10.5, 10.9, 11.4 and 17.8.
  a.least = 2;
  a.scale_log2 = scale * 1.4426950408889634f;
  uint8_t* p = static_cast<uint8_t*>(ws);
  a.notes = reinterpret_cast<PartialNote*>(p);
  a.ml = reinterpret_cast<float2*>(p + z.notes);
  a.o = reinterpret_cast<float*>(p + z.notes + z.ml);
  if (elem == 10) return z.dp == 64 ? launch_rows<__half, 64>(a, s) : launch_rows<__half, 128>(a, s);
  return z.dp == 64 ? launch_rows<__nv_bfloat16, 64>(a, s) : launch_rows<__nv_bfloat16, 128>(a, s);
}

}  // namespace k
}  // namespace sb
