// A mixture-of-experts layer for a few tokens:
//   l = x R^T,  s = softmax(l) or 1 / (1 + e^-l),  the top_k largest s (+ selection bias), share_e = s_e (/ their sum) scale
//   y = sum over the chosen e of share_e D_e (act(G_e x) * (U_e x))
//
// Few tokens read each chosen expert's weights for a handful of columns: the weights' bytes bound it. The products
// go to the tensor core (mma m16n8k16, fp32 accumulators) with the weights as the 16-row operand and up to 8 tokens
// as its columns, so that a token more costs next to nothing. Its inputs' order in k does not matter as long as both
// operands have the same, so a lane takes 8 neighbouring inputs of a row as its part of two products: weights come as
// they lie in memory, in 16-byte pieces that only the lane that copied them reads (a cp.async ring per warp, without
// barriers, that runs on over the ends of tiles).
// A tile of the first product holds 8 rows of G and the same 8 of U: a lane has gate and input of one feature.
//
// Four kernels in a chain, each launched while the one before it runs: the router's dot products and the choice, a cluster
// per token; the first product over (expert, features), its k split over a CTA's warps; the second over (expert, outputs,
// part of k) into partial sums, whose weights are on their way before the first has ended; their sum in the order of a
// token's experts. No atomics decide an order: results repeat. (All of it in one cooperative launch took 33 us where the chain
// took 27, for a token through 8 of 128 experts of 2048 x 768: such a launch and its three barriers cost 8 us, these four
// kernels 4.)
// Measured: 13 tokens through 6 of 64 experts of 4096 x 1400 in fp16 (1.6 GB) 266 us, 6.0 TB/s; one token (75 MB) 29 us,
// of which the router and the choice take 6, the lists 1, the products 18; 200 tokens of 32 experts (0.4 GB) 130 to 138 us.
//
// The router's sums, scores and their order are in fp64: a choice between experts whose scores are next to each other
// hangs on it. Hidden values are two numbers of the weights' type, the second product's operands (see below);
// all else stays in fp32.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "decoder.h"

namespace sb {
namespace k {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStages = 5;          // steps of a ring
constexpr int kBlock = 64;          // inputs of a step
constexpr int kMostExperts = 512;   // a lane has 16 scores
constexpr int kRouteCtas = 8, kRouteThreads = 512;   // of a token's cluster, at most

struct Entry { int expert, first, count; };   // up to 8 NT places of the list, of one expert

struct MoEArgs {
  MoEView w;
  const void* x;
  void* y;
  int64_t xs, ys;
  int tokens, rows;        // rows: tokens * top_k
  int entries;             // room for them
  int splits;              // of the second product's k
  int* chosen;             // [rows]
  float* share;            // [rows]
  void* hidden;            // [2][rows][inner]: values in the weights' type, and kRest times what they lost
  float* partial;          // [splits][rows][width]
};

template <typename T> struct Op;
template <> struct Op<__half> {
  static __device__ __forceinline__ float2 both(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static constexpr float kMost = 65504.f, kRest = 2048.f;
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Op<__nv_bfloat16> {
  static __device__ __forceinline__ float2 both(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
  static constexpr float kMost = 3.38953139e38f, kRest = 256.f;
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {   // zeros where it is not
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// A score as an integer of the same order, NaN below all and 0 for none. In 64 bits: scores that fp32 does not tell apart, more
// of them beside a large bias, would go by the expert's number.
__device__ __forceinline__ unsigned long long ordered(double v) {
  if (v != v) return 1ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
  return b >> 63 ? ~b : b | 1ull << 63;
}

// One dot product of the router, by a warp.
template <typename T>
__device__ __forceinline__ double router_dot(const MoEArgs& a, int t, int e, int lane) {
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + t * a.xs;
  double sum = 0;
  if (a.w.router_elem == 1) {
    const float* r = static_cast<const float*>(a.w.router) + e * a.w.router_row;
#pragma unroll 4
    for (int k = lane * 8; k < a.w.width; k += 256) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + k);
      const float4 p = *reinterpret_cast<const float4*>(r + k), q = *reinterpret_cast<const float4*>(r + k + 4);
      const float2 v0 = Op<T>::both(v.x), v1 = Op<T>::both(v.y), v2 = Op<T>::both(v.z), v3 = Op<T>::both(v.w);
      sum += double(v0.x) * p.x + double(v0.y) * p.y + double(v1.x) * p.z + double(v1.y) * p.w;
      sum += double(v2.x) * q.x + double(v2.y) * q.y + double(v3.x) * q.z + double(v3.y) * q.w;
    }
  } else {
    const uint16_t* r = static_cast<const uint16_t*>(a.w.router) + e * a.w.router_row;
#pragma unroll 8
    for (int k = lane * 8; k < a.w.width; k += 256) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + k), q = *reinterpret_cast<const uint4*>(r + k);
      const float2 v0 = Op<T>::both(v.x), v1 = Op<T>::both(v.y), v2 = Op<T>::both(v.z), v3 = Op<T>::both(v.w);
      const float2 q0 = Op<T>::both(q.x), q1 = Op<T>::both(q.y), q2 = Op<T>::both(q.z), q3 = Op<T>::both(q.w);
      // products of 16-bit numbers are exact in fp32 (converted once, not twice: one token of 512 experts 39 us, not 46)
      sum += (double(v0.x * q0.x) + double(v0.y * q0.y)) + (double(v1.x * q1.x) + double(v1.y * q1.y));
      sum += (double(v2.x * q2.x) + double(v2.y * q2.y)) + (double(v3.x * q3.x) + double(v3.y * q3.y));
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
  return sum;
}

// What only some layers need, in fp64 (not inline: the choice is a chain that runs once, and waits for its instructions):
// the largest logit and the sum of e^(l - top) over all experts,
template <int J> __device__ __noinline__ void sum_scores(const double (&v)[J], int experts, int lane, double& top, double& all) {
  double t = -INFINITY, a = 0;
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (j * 32 + lane < experts) t = fmax(t, v[j]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) t = fmax(t, __shfl_xor_sync(~0u, t, d));
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (j * 32 + lane < experts) a += exp(v[j] - t);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) a += __shfl_xor_sync(~0u, a, d);
  top = t, all = a;
}
// and the order of score + bias.
template <int J>
__device__ __noinline__ void bias_keys(unsigned long long (&key)[J], const double (&v)[J], const MoEView& w, int lane, double top, double all) {
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = j * 32 + lane;
    if (e < w.experts) key[j] = ordered((w.softmax ? exp(v[j] - top) / all : 1.0 / (1.0 + exp(-v[j]))) + double(w.selection_bias[e]));
  }
}

// The experts of a token and their shares from its logits, by a warp; equal scores go to the lower expert. J: scores per
// lane.
template <int J>
__device__ __forceinline__ void choose(const MoEView& w, const double* l, int lane, int* chosen, float* share) {
  double v[J];
#pragma unroll
  for (int j = 0; j < J; ++j) v[j] = j * 32 + lane < w.experts ? l[j * 32 + lane] : 0.0;
  unsigned long long key[J];
#pragma unroll
  for (int j = 0; j < J; ++j) key[j] = j * 32 + lane < w.experts ? ordered(v[j]) : 0ull;
  double top = 0, all = 0;
  const bool biased = w.selection_bias != nullptr;
  if (w.softmax && (biased || !w.normalize)) sum_scores<J>(v, w.experts, lane, top, all);
  if (biased) bias_keys<J>(key, v, w, lane, top, all);
  int mine = 0;          // lane r: the r-th chosen
  for (int r = 0; r < w.top_k; ++r) {
    unsigned long long best = key[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < J; ++j)
      if (key[j] > best) best = key[j], at = j;
    const uint32_t upper = uint32_t(best >> 32), lower = uint32_t(best);
    const bool first = upper == __reduce_max_sync(~0u, upper);
    const uint32_t rest = __reduce_max_sync(~0u, first ? lower : 0u);
    const uint32_t e = __reduce_min_sync(~0u, first && lower == rest ? at * 32 + lane : ~0u);
    if ((e & 31) == uint32_t(lane)) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (e >> 5 == uint32_t(j)) key[j] = 0;
    }
    if (lane == r) mine = int(e);
  }
  const double z = l[mine];
  // Shares that are normalized are quotients, whatever the scores are multiplied by: a factor that brings the largest of the
  // chosen near 1 keeps them within fp32's range. Its logit is the first chosen's, but where a bias has chosen.
  double high = top;
  if (w.normalize) {
    high = biased && lane >= w.top_k ? -INFINITY : z;
    if (biased) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) high = fmax(high, __shfl_xor_sync(~0u, high, d));
    }
    high = __shfl_sync(~0u, high, 0);
  }
  float s;
  if (w.softmax) {
    s = expf(float(z - high));
  } else {   // e^-c / (1 + e^-z), with c the largest logit where that is below 0
    const double c = w.normalize ? fmin(high, 0.0) : 0.0;
    s = 1.f / (expf(float(c)) + expf(float(c - z)));
  }
  if (lane >= w.top_k) s = 0.f;
  if (w.normalize) {
    float sum = s;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    s /= sum;
  } else if (w.softmax) {
    s /= float(all);
  }
  if (lane < w.top_k) {
    chosen[lane] = mine;
    share[lane] = s * w.scale;
  }
}

template <typename T>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const __grid_constant__ MoEArgs a) {
  __shared__ double logits[kMostExperts];   // of the cluster's first CTA
  asm volatile("griddepcontrol.launch_dependents;");
  const auto cluster = cooperative_groups::this_cluster();
  const int ctas = int(cluster.num_blocks()), t = blockIdx.x / ctas, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double* to = cluster.map_shared_rank(logits, 0);
  asm volatile("barrier.cluster.arrive.relaxed.aligned;");   // the first CTA has begun, when the wait below is over
  bool begun = false;
  for (int e = warp * ctas + int(cluster.block_rank()); e < a.w.experts; e += ctas * (kRouteThreads / 32)) {
    const double v = router_dot<T>(a, t, e, lane);
    if (!begun) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    begun = true;
    if (lane == 0) to[e] = v;
  }
  if (!begun) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  cluster.sync();
  if (cluster.block_rank() == 0 && warp == 0) {
    int* chosen = a.chosen + t * a.w.top_k;
    float* share = a.share + t * a.w.top_k;
    if (a.w.experts <= 128) choose<4>(a.w, logits, lane, chosen, share);
    else choose<kMostExperts / 32>(a.w, logits, lane, chosen, share);
  }
}

// What a CTA knows of the step's rows (t * top_k + r: the r-th expert of token t), in shared memory.
struct Lists {
  Entry* entry;        // [entries]
  int* number;         // [kWarps][experts] rows of an expert among a warp's quarter of them, then places before those
  int* chosen;         // [rows]
  int* count;          // entries in use
  uint16_t* row;       // the list: [rows], by expert
  uint16_t* place;     // [rows] among its expert's of its quarter
};
__host__ __device__ inline size_t lists_bytes(int experts, int entries, int rows) {
  return size_t(entries) * sizeof(Entry) + size_t(experts) * kWarps * 4 + size_t(rows) * 8 + 32;
}

// The rows by expert, in their order: all CTAs have to divide an expert's rows among its entries alike.
template <int NT> __device__ __forceinline__ Lists make_lists(const MoEArgs& a, uint8_t* p, int tid) {
  Lists at;
  const int experts = a.w.experts, lane = tid & 31, warp = tid >> 5;
  at.entry = reinterpret_cast<Entry*>(p), p += a.entries * sizeof(Entry);
  at.number = reinterpret_cast<int*>(p), p += size_t(experts) * kWarps * 4;
  at.chosen = reinterpret_cast<int*>(p), p += size_t(a.rows) * 4;
  at.count = reinterpret_cast<int*>(p), p += 32;   // and the warps' sums
  at.row = reinterpret_cast<uint16_t*>(p), p += size_t(a.rows) * 2;
  at.place = reinterpret_cast<uint16_t*>(p);
  if (a.tokens == 1) {   // an entry per row, in any order
    if (tid < a.rows) at.entry[tid] = {__ldcg(a.chosen + tid), tid, 1}, at.row[tid] = uint16_t(tid);
    if (tid == 0) *at.count = a.rows;
    __syncthreads();
    return at;
  }
  for (int i = tid; i < experts * kWarps; i += kThreads) at.number[i] = 0;
  for (int i = tid; i < a.rows; i += kThreads) at.chosen[i] = __ldcg(a.chosen + i);
  __syncthreads();
  const int quarter = (a.rows + kWarps * 32 - 1) / (kWarps * 32) * 32;
  int* number = at.number + warp * experts;
  for (int i0 = warp * quarter; i0 < min((warp + 1) * quarter, a.rows); i0 += 32) {
    const int i = i0 + lane, e = i < a.rows ? at.chosen[i] : -1 - lane;
    const uint32_t same = __match_any_sync(~0u, e), lower = same & ((1u << lane) - 1);
    if (e >= 0) {
      const int before = number[e];
      at.place[i] = uint16_t(before + __popc(lower));
      __syncwarp(same);
      if (lower == 0) number[e] = before + __popc(same);
    }
    __syncwarp();
  }
  __syncthreads();
  // four experts per thread: where their rows begin, and their entries
  constexpr int kEach = kMostExperts / kThreads;
  int n[kEach], rows = 0, entries = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = tid * kEach + i;
    n[i] = 0;
    if (e < experts)
      for (int w = 0; w < kWarps; ++w) n[i] += at.number[w * experts + e];
    rows += n[i], entries += (n[i] + 8 * NT - 1) / (8 * NT);
  }
  int both = rows << 16 | entries;   // each below 2^15
  const int own = both;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int before = __shfl_up_sync(~0u, both, d);
    if (lane >= d) both += before;
  }
  if (lane == 31) at.count[1 + warp] = both;
  __syncthreads();
  for (int w = 0; w < warp; ++w) both += at.count[1 + w];
  if (tid == kThreads - 1) *at.count = both & 0xffff;
  rows = (both - own) >> 16, entries = (both - own) & 0xffff;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = tid * kEach + i;
    for (int k = 0; k < n[i]; k += 8 * NT) at.entry[entries++] = {e, rows + k, min(8 * NT, n[i] - k)};
    if (e < experts) {
      int first = rows;
      for (int w = 0; w < kWarps; ++w) {
        const int m = at.number[w * experts + e];
        at.number[w * experts + e] = first;
        first += m;
      }
    }
    rows += n[i];
  }
  __syncthreads();
  for (int i = tid; i < a.rows; i += kThreads) at.row[at.number[i / quarter * experts + at.chosen[i]] + at.place[i]] = uint16_t(i);
  __syncthreads();
  return at;
}

__device__ __forceinline__ float activated(int gelu, float gate, float up) {
  return (gelu ? 0.5f * gate * (1.f + erff(gate * 0.70710678f)) : gate / (1.f + expf(-gate))) * up;
}

// A hidden value goes to the second product as two operands: rounded to the type, and kRest times the rest of it, which keeps
// fp16's rests normal numbers. Together they have the bits that the second product's fp32 sums can make use of, 16 in bf16
// and 22 in fp16; rounded once, they added half as much again to the error of the results. (Beyond the type's largest
// number the rest is infinite, and so is the result.)
template <typename T> __device__ __forceinline__ void store_hidden(const MoEArgs& a, int row, int feature, float v) {
  T* to = static_cast<T*>(a.hidden) + int64_t(row) * a.w.inner + feature;
  const T whole = Op<T>::round(fminf(fmaxf(v, -Op<T>::kMost), Op<T>::kMost));
  to[0] = whole;
  to[int64_t(a.rows) * a.w.inner] = Op<T>::round((v - Op<T>::widen(whole)) * Op<T>::kRest);
}

// The sums over both operands. (One that is infinite by its weights has no rest: infinities of another sign would make it NaN.)
template <typename T> __device__ __forceinline__ float joined(float whole, float rest) {
  return isfinite(whole) ? fmaf(rest, 1.f / Op<T>::kRest, whole) : whole;
}

// The two products, for up to 8 rows of an expert. Units: (entry, tile of 8 features or 16 outputs, part of k); a CTA takes
// every gridDim.x-th, its warps every kWarps-th block of k.
template <typename T, bool kFirst>
struct Product {
  static constexpr int kTile = kFirst ? 8 : 16, kStage = 2048;   // bytes of a step: 16 rows of 64 inputs
  static constexpr int kSets = kFirst ? 1 : 2;                   // of columns: hidden values and their rests
  const MoEArgs& a;
  const Lists& at;
  const uint32_t ring;   // this warp's
  float* sums;           // [2][kWarps][4][32]
  const int lane, warp, g, t;
  int units, tiles, parts, blocks, depth, out_rows;   // blocks of k in a part; depth: k; out_rows: rows of the weights (of each half)
  int64_t expert_stride, row_stride, second;          // second: from a row to the one that is 8 further in the tile
  const uint16_t* weights;
  int copy_unit, copy_block, copy_end;   // the next step to copy
  const uint16_t* copy_from;
  bool copy_second;                      // whether the tile has its second 8 rows
  int stage_in, stage_out;

  __device__ __forceinline__ Product(const MoEArgs& args, const Lists& lists, uint32_t ring_at, float* sums_at)
      : a(args), at(lists), ring(ring_at), sums(sums_at), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), g(lane >> 2), t(lane & 3) {
    depth = kFirst ? a.w.width : a.w.inner;
    out_rows = kFirst ? a.w.inner : a.w.width;
    parts = kFirst ? 1 : a.splits;
    blocks = ((depth + kBlock - 1) / kBlock + parts - 1) / parts;
    tiles = (out_rows + kTile - 1) / kTile;
    units = *at.count * tiles * parts;
    expert_stride = kFirst ? a.w.up_expert : a.w.down_expert;
    row_stride = kFirst ? a.w.up_row : a.w.down_row;
    second = (kFirst ? int64_t(a.w.inner) : 8) * row_stride;
    weights = static_cast<const uint16_t*>(kFirst ? a.w.gate_up : a.w.down);
    stage_in = stage_out = 0;
    copy_unit = int(blockIdx.x) - int(gridDim.x);
    next_unit();
  }
  struct Unit { int entry, first, part; };
  __device__ __forceinline__ Unit unit(int u) const {
    Unit v;
    const int e = u / parts;
    v.part = u - e * parts;
    v.entry = e / tiles;
    v.first = (e - v.entry * tiles) * kTile;
    return v;
  }
  __device__ __forceinline__ int end_of(const Unit& v) const { return min((v.part + 1) * blocks, (depth + kBlock - 1) / kBlock); }

  __device__ __forceinline__ void next_unit() {   // to the next unit in which this warp has a step
    do {
      copy_unit += int(gridDim.x);
      if (copy_unit >= units) return;
      const Unit v = unit(copy_unit);
      copy_block = v.part * blocks + warp;
      copy_end = end_of(v);
      copy_from = weights + at.entry[v.entry].expert * expert_stride + (v.first + g) * row_stride + 8 * t;
      copy_second = kFirst || v.first + 8 < out_rows;   // (features and outputs come in eights)
    } while (copy_block >= copy_end);
  }
  __device__ __forceinline__ void copy_step() {
    if (copy_unit < units) {
      const uint32_t to = ring + stage_in * kStage + lane * 16;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = copy_block * kBlock + h * 32;
          const bool there = (r == 0 || copy_second) && k + 8 * t < depth;
          copy16(to + (r * 2 + h) * 512, there ? copy_from + r * second + k : weights, there);
        }
      copy_block += kWarps;
      if (copy_block >= copy_end) next_unit();
    }
    commit();
    stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
  }
  __device__ __forceinline__ void fill() {
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy_step();
  }

  __device__ __forceinline__ void run() {
    int turn = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const Unit v = unit(u);
      const Entry en = at.entry[v.entry];
      const uint16_t* rows = at.row + en.first;
      const uint16_t* column = nullptr;   // of the lane's token
      if (g < en.count)
        column = kFirst ? static_cast<const uint16_t*>(a.x) + rows[g] / a.w.top_k * a.xs : static_cast<const uint16_t*>(a.hidden) + int64_t(rows[g]) * a.w.inner;
      auto fetch = [&](uint4 (&b)[kSets][2], int block) {
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = block * kBlock + h * 32 + 8 * t;
            b[s][h] = make_uint4(0, 0, 0, 0);
            if (column != nullptr && k < depth) b[s][h] = *reinterpret_cast<const uint4*>(column + s * (int64_t(a.rows) * a.w.inner) + k);
          }
      };
      float d[kSets][4] = {};
      auto step = [&](const uint4 (&b)[kSets][2]) {
        wait<kStages - 2>();
        const uint32_t from = ring + stage_out * kStage + lane * 16;
        stage_out = stage_out + 1 == kStages ? 0 : stage_out + 1;
        uint4 w[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) w[r][h] = shared16(from + (r * 2 + h) * 512);
        copy_step();   // into the stage read in the step before
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int s = 0; s < kSets; ++s) {
            Op<T>::mma(d[s], w[0][h].x, w[1][h].x, w[0][h].y, w[1][h].y, b[s][h].x, b[s][h].y);
            Op<T>::mma(d[s], w[0][h].z, w[1][h].z, w[0][h].w, w[1][h].w, b[s][h].z, b[s][h].w);
          }
      };
      // Columns are fetched a step ahead, into registers of their own by turns (a copy between them would wait for them).
      const int end = end_of(v);
      int block = v.part * blocks + warp;
      uint4 even[kSets][2], odd[kSets][2];
      if (block < end) fetch(even, block);
      while (block < end) {
        if (block + kWarps < end) fetch(odd, block + kWarps);
        step(even);
        block += kWarps;
        if (block >= end) break;
        if (block + kWarps < end) fetch(even, block + kWarps);
        step(odd);
        block += kWarps;
      }
      // The warps' sums meet; two buffers in turn, so that one barrier is enough.
      float* all = sums + turn * kWarps * 128;
      turn ^= 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) all[warp * 128 + i * 32 + lane] = kFirst ? d[0][i] : joined<T>(d[0][i], d[kSets - 1][i]);
      __syncthreads();
      auto total = [&](int q) { return all[q] + all[128 + q] + all[256 + q] + all[384 + q]; };
      static_assert(kWarps == 4, "the sum above");
      const int l = threadIdx.x & 31, q = threadIdx.x >> 5;   // a value of the tile per thread, or a pair of them
      const int c = (l & 3) * 2 + (q & 1);
      if (kFirst) {
        if (q < 2 && c < en.count) store_hidden<T>(a, rows[c], v.first + (l >> 2), activated(a.w.gelu, total(q * 32 + l), total((q + 2) * 32 + l)));
      } else {
        const int r = v.first + (q >> 1) * 8 + (l >> 2);
        if (c < en.count && r < out_rows) a.partial[(int64_t(v.part) * a.rows + rows[c]) * out_rows + r] = total(q * 32 + l);
      }
    }
  }
};

// The same for experts of many tokens, 32 at a time: there the columns weigh as much as the weights, so a CTA's warps share
// them (in shared memory, swizzled by 16-byte pieces) and have rows of their own, over all of k.
template <typename T, bool kFirst>
struct WideProduct {
  // kRing: steps of the ring. With twice the columns the second product's is shorter, so that two CTAs share an SM beside their
  // lists (256 tokens through 8 of 64 experts of 1024 x 512: 118 us, 131 with four steps; 200 of 32 experts 129 and 133).
  static constexpr int NT = 4, MT = 2, kRing = kFirst ? 4 : 3;
  static constexpr int kWarpRows = kFirst ? 8 * MT : 16 * MT, kTile = kWarps * kWarpRows, kApart = kFirst ? 8 : 16;
  static constexpr int kSets = kFirst ? 1 : 2, kColumns = NT * 8 * 128;   // of columns; bytes of a set
  static constexpr int kStage = kWarps * MT * 2048 + kSets * kColumns;
  const MoEArgs& a;
  const Lists& at;
  const uint32_t ring;
  const int tid, lane, warp, g, t;
  int units, tiles, parts, blocks, depth, out_rows;
  int64_t expert_stride, row_stride, second;
  const uint16_t* weights;
  int copy_unit, copy_block, copy_end;
  const uint16_t* copy_from;
  const uint16_t* copy_column;   // of the token that this thread copies, or null
  uint32_t copy_there;
  int stage_in, stage_out;

  __device__ __forceinline__ WideProduct(const MoEArgs& args, const Lists& lists, uint32_t ring_at)
      : a(args), at(lists), ring(ring_at), tid(threadIdx.x), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), g(lane >> 2), t(lane & 3) {
    depth = kFirst ? a.w.width : a.w.inner;
    out_rows = kFirst ? a.w.inner : a.w.width;
    parts = kFirst ? 1 : a.splits;
    blocks = ((depth + kBlock - 1) / kBlock + parts - 1) / parts;
    tiles = (out_rows + kTile - 1) / kTile;
    units = *at.count * tiles * parts;
    expert_stride = kFirst ? a.w.up_expert : a.w.down_expert;
    row_stride = kFirst ? a.w.up_row : a.w.down_row;
    second = (kFirst ? int64_t(a.w.inner) : 8) * row_stride;
    weights = static_cast<const uint16_t*>(kFirst ? a.w.gate_up : a.w.down);
    stage_in = stage_out = 0;
    copy_unit = int(blockIdx.x) - int(gridDim.x);
    next_unit();
  }
  struct Unit { int entry, first, part, begin, end; };
  __device__ __forceinline__ Unit unit(int u) const {   // entries innermost: those of one expert read its weights together
    Unit v;
    const int e = u / *at.count;
    v.entry = u - e * *at.count;
    v.part = e % parts;
    v.first = e / parts * kTile;
    v.begin = v.part * blocks;
    v.end = min(v.begin + blocks, (depth + kBlock - 1) / kBlock);
    return v;
  }
  __device__ __forceinline__ void next_unit() {
    do {
      copy_unit += int(gridDim.x);
      if (copy_unit >= units) return;
      const Unit v = unit(copy_unit);
      const Entry en = at.entry[v.entry];
      copy_block = v.begin, copy_end = v.end;
      copy_from = weights + en.expert * expert_stride + (v.first + warp * kWarpRows + g) * row_stride + 8 * t;
      copy_there = 0;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int r = v.first + warp * kWarpRows + m * kApart + g;
        if (r < out_rows) copy_there |= 1u << (2 * m);
        if (r + (kFirst ? 0 : 8) < out_rows) copy_there |= 2u << (2 * m);
      }
      copy_column = nullptr;
      if (tid / 4 < en.count) {
        const int row = at.row[en.first + tid / 4];
        copy_column = kFirst ? static_cast<const uint16_t*>(a.x) + row / a.w.top_k * a.xs : static_cast<const uint16_t*>(a.hidden) + int64_t(row) * a.w.inner;
      }
    } while (copy_block >= copy_end);
  }
  __device__ __forceinline__ void copy_step() {
    if (copy_unit < units) {
      const uint32_t stage = ring + stage_in * kStage, to = stage + warp * (MT * 2048) + lane * 16;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = copy_block * kBlock + h * 32;
            const bool there = (copy_there >> (2 * m + r) & 1) && k + 8 * t < depth;
            copy16(to + ((m * 2 + r) * 2 + h) * 512, there ? copy_from + m * kApart * row_stride + r * second + k : weights, there);
          }
      const int token = tid / 4;   // two of its 8 pieces
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = (tid % 4) * 2 + i, k = copy_block * kBlock + c * 8;
        const bool there = copy_column != nullptr && k < depth;
#pragma unroll
        for (int s = 0; s < kSets; ++s)
          copy16(stage + kWarps * MT * 2048 + s * kColumns + token * 128 + ((c ^ (token & 7)) * 16),
                 there ? copy_column + s * (int64_t(a.rows) * a.w.inner) + k : weights, there);
      }
      if (++copy_block >= copy_end) next_unit();
    }
    commit();
    stage_in = stage_in + 1 == kRing ? 0 : stage_in + 1;
  }
  __device__ __forceinline__ void run() {
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) copy_step();
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const Unit v = unit(u);
      const Entry en = at.entry[v.entry];
      const int used = (en.count + 7) / 8;
      float d[kSets][NT][MT][4] = {};
      for (int block = v.begin; block < v.end; ++block) {
        wait<kRing - 2>();
        __syncthreads();   // all copies of this step are there, and all have read the step before
        const uint32_t stage = ring + stage_out * kStage, from = stage + warp * (MT * 2048) + lane * 16;
        stage_out = stage_out + 1 == kRing ? 0 : stage_out + 1;
        uint4 w[MT][2][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[m][r][h] = shared16(from + ((m * 2 + r) * 2 + h) * 512);
        copy_step();   // into the stage read in the step before
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n >= used) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int s = 0; s < kSets; ++s) {
              const uint4 b = shared16(stage + kWarps * MT * 2048 + s * kColumns + (n * 8 + g) * 128 + (((h * 4 + t) ^ g) * 16));
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                Op<T>::mma(d[s][n][m], w[m][0][h].x, w[m][1][h].x, w[m][0][h].y, w[m][1][h].y, b.x, b.y);
                Op<T>::mma(d[s][n][m], w[m][0][h].z, w[m][1][h].z, w[m][0][h].w, w[m][1][h].w, b.z, b.w);
              }
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n >= used) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = n * 8 + t * 2 + i;
          if (c >= en.count) continue;
          const int row = at.row[en.first + c];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const int r = v.first + warp * kWarpRows + m * kApart + g;
            if (kFirst) {
              if (r < out_rows) store_hidden<T>(a, row, r, activated(a.w.gelu, d[0][n][m][i], d[0][n][m][i + 2]));
            } else {
              float* to = a.partial + (int64_t(v.part) * a.rows + row) * out_rows + r;
              auto both = [&](int j) { return joined<T>(d[0][n][m][j], d[kSets - 1][n][m][j]); };
              if (r < out_rows) to[0] = both(i);
              if (r + 8 < out_rows) to[8] = both(i + 2);
            }
          }
        }
      }
    }
    wait<0>();
  }
};

constexpr int kSums = 2 * kWarps * 128 * 4;   // of the warps, twice
template <typename T, int NT, bool kFirst> constexpr int ring_bytes() {
  if constexpr (NT == 1) return kWarps * kStages * 2048;
  else return WideProduct<T, kFirst>::kRing * WideProduct<T, kFirst>::kStage;
}
template <typename T, int NT, bool kFirst>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 2) product_kernel(const __grid_constant__ MoEArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kHeld = ring_bytes<T, NT, kFirst>() + (NT == 1 ? kSums : 0);
  // The choice is there: for the first product once the router has ended; the second is launched after that, as the first
  // lets it begin behind its own wait.
  if (kFirst) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Lists at = make_lists<NT>(a, smem + kHeld, threadIdx.x);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  if constexpr (NT == 1) {
    Product<T, kFirst> product(a, at, ring + (threadIdx.x >> 5) * kStages * 2048, reinterpret_cast<float*>(smem + ring_bytes<T, NT, kFirst>()));
    product.fill();   // weights, while the first product finishes the hidden values
    if (!kFirst) asm volatile("griddepcontrol.wait;" ::: "memory");
    product.run();
    wait<0>();
  } else {
    WideProduct<T, kFirst> product(a, at, ring);
    if (!kFirst) asm volatile("griddepcontrol.wait;" ::: "memory");
    product.run();
  }
}

// y of four outputs of a token per thread
template <typename T>
__global__ void __launch_bounds__(kThreads) combine_kernel(const __grid_constant__ MoEArgs a) {
  const int quads = a.w.width / 4, top_k = a.w.top_k;
  const int i = blockIdx.x * kThreads + threadIdx.x;
  const int t = i / quads, h = (i - t * quads) * 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (t >= a.tokens) return;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* p = a.partial + int64_t(t) * top_k * a.w.width + h;
  for (int r0 = 0; r0 < top_k; r0 += 4) {   // loads in flight together
    float4 v[4];
    float share[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r0 + r < top_k) {
        v[r] = __ldcg(reinterpret_cast<const float4*>(p + int64_t(r0 + r) * a.w.width));
        share[r] = __ldcg(a.share + t * top_k + r0 + r);
      }
    for (int j = 1; j < a.splits; ++j) {
      float4 u[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r0 + r < top_k) u[r] = __ldcg(reinterpret_cast<const float4*>(p + (int64_t(j) * a.rows + r0 + r) * a.w.width));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r0 + r < top_k) v[r].x += u[r].x, v[r].y += u[r].y, v[r].z += u[r].z, v[r].w += u[r].w;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r0 + r < top_k) y.x += share[r] * v[r].x, y.y += share[r] * v[r].y, y.z += share[r] * v[r].z, y.w += share[r] * v[r].w;
  }
  alignas(8) T out[4] = {Op<T>::round(y.x), Op<T>::round(y.y), Op<T>::round(y.z), Op<T>::round(y.w)};
  *reinterpret_cast<uint2*>(static_cast<T*>(a.y) + t * a.ys + h) = *reinterpret_cast<const uint2*>(out);
}

// Sizes of one launch over up to `tokens` tokens.
struct Sizes {
  int tokens, entries, splits, columns;
  size_t chosen, hidden, partial, total;
};
Sizes sizes(const MoEView& w, int64_t tokens) {
  Sizes z;
  z.tokens = int(std::min<int64_t>(std::max<int64_t>(tokens, 1), std::min(256, 2048 / w.top_k)));
  const int rows = z.tokens * w.top_k;
  // Columns of a product: 8 where an expert has few tokens on average; an expert that has more is read again (from L2, as
  // its entries are near each other in time). 8 of 128 experts of 2048 x 768, 4 tokens each on average: 219 us with 8
  // columns, 240 with 32; 6 tokens 250 and 255, 8 tokens 306 and 262. (6 of 64: 9 tokens 156 and 149.)
  z.columns = z.tokens <= 8 || rows <= 6 * w.experts ? 8 : 32;
  z.entries = std::min(w.experts, rows) + rows / z.columns;
  // Parts of the second product's k, of 1024 inputs or more, until (expert, tile, part) triples are many for every CTA (64
  // tokens through 2 of 8 experts of 1024 x 4096 75 us, in one part 138, in parts of 512 79; half or twice as many
  // triples: within 2 in 100)
  const int tile = z.columns == 8 ? 16 : 32 * kWarps;
  const int64_t units = int64_t(std::min(w.experts, rows)) * ((w.width + tile - 1) / tile), enough = z.columns == 8 ? 4096 : 1024;
  z.splits = 1;
  while (z.splits < 8 && units * z.splits < enough && w.inner / (z.splits * 2) >= 1024) z.splits *= 2;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  z.chosen = up(size_t(rows) * 4);
  z.hidden = up(size_t(rows) * w.inner * 4);
  z.partial = up(size_t(z.splits) * rows * w.width * 4);
  z.total = 2 * z.chosen + z.hidden + z.partial;
  return z;
}

cudaError_t enqueue(void (*kernel)(MoEArgs), const MoEArgs& a, int64_t grid, int threads, size_t smem, int cluster, bool after, cudaStream_t s) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(unsigned(grid)), c.blockDim = dim3(unsigned(threads)), c.dynamicSmemBytes = smem, c.stream = s;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster) at[n].id = cudaLaunchAttributeClusterDimension, at[n].val.clusterDim = {unsigned(cluster), 1, 1}, ++n;
  if (after) at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[n].val.programmaticStreamSerializationAllowed = 1, ++n;
  c.attrs = at, c.numAttrs = unsigned(n);
  return cudaLaunchKernelEx(&c, kernel, a);
}

template <typename T, int NT, bool kFirst>
cudaError_t product(const MoEArgs& a, int sms, cudaStream_t s) {
  const size_t smem = size_t(ring_bytes<T, NT, kFirst>()) + (NT == 1 ? kSums : 0) + lists_bytes(a.w.experts, a.entries, a.rows);
  const auto kernel = product_kernel<T, NT, kFirst>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e != cudaSuccess) return e;
  const int64_t each = std::min<int64_t>(NT == 1 ? 4 : 2, 227 * 1024 / (smem + 1024));
  const int rows = kFirst ? a.w.inner : a.w.width, tile = (kFirst ? 8 : 16) * (NT == 1 ? 1 : 2 * kWarps);
  const int64_t units = int64_t(a.entries) * ((rows + tile - 1) / tile) * (kFirst ? 1 : a.splits);   // at most
  return enqueue(kernel, a, std::min(units, std::max<int64_t>(each, 1) * sms), kThreads, smem, 0, true, s);
}

template <typename T>
cudaError_t launch(const MoEArgs& a, int columns, int sms, cudaStream_t s) {
  int ctas = 1;   // a warp per expert while that fits the card (200 tokens of 32 experts by 8 CTAs each: 20 us)
  while (ctas < kRouteCtas && ctas * (kRouteThreads / 32) < a.w.experts && int64_t(a.tokens) * ctas <= 2 * sms) ctas *= 2;
  cudaError_t e = enqueue(route_kernel<T>, a, int64_t(a.tokens) * ctas, kRouteThreads, 0, ctas, false, s);
  if (e == cudaSuccess) e = columns == 8 ? product<T, 1, true>(a, sms, s) : product<T, 4, true>(a, sms, s);
  if (e == cudaSuccess) e = columns == 8 ? product<T, 1, false>(a, sms, s) : product<T, 4, false>(a, sms, s);
  if (e != cudaSuccess) return e;
  return enqueue(combine_kernel<T>, a, (int64_t(a.tokens) * (a.w.width / 4) + kThreads - 1) / kThreads, kThreads, 0, 0, true, s);
}

}  // namespace

size_t moe_workspace(const MoEView& w, int64_t tokens) {
  const Sizes z = sizes(w, tokens);
  return std::max(z.total, sizes(w, tokens % z.tokens).total);
}

cudaError_t moe(const MoEView& w, const void* x, int64_t xs, void* y, int64_t ys, int64_t tokens, void* ws, int sms, cudaStream_t s) {
  // More tokens than a launch takes go through in pieces.
  const Sizes most = sizes(w, tokens);
  for (int64_t t0 = 0; t0 < tokens; t0 += most.tokens) {
    const Sizes z = sizes(w, std::min<int64_t>(most.tokens, tokens - t0));
    MoEArgs a;
    a.w = w;
    a.x = static_cast<const uint16_t*>(x) + t0 * xs, a.y = static_cast<uint16_t*>(y) + t0 * ys, a.xs = xs, a.ys = ys;
    a.tokens = z.tokens, a.rows = z.tokens * w.top_k, a.entries = z.entries, a.splits = z.splits;
    uint8_t* p = static_cast<uint8_t*>(ws);
    a.chosen = reinterpret_cast<int*>(p), p += z.chosen;
    a.share = reinterpret_cast<float*>(p), p += z.chosen;
    a.hidden = p, p += z.hidden;
    a.partial = reinterpret_cast<float*>(p);
    const cudaError_t e = w.elem == 10 ? launch<__half>(a, z.columns, sms, s) : launch<__nv_bfloat16>(a, z.columns, sms, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace k
}  // namespace sb
