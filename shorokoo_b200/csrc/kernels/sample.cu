// The next token of each row of logits, from a given random number:
//   w_i = exp((l_i - max) / T); kept are w_i >= min_p, of these the top_k largest, of these the fewest largest whose sum is
//   at least top_p of theirs (equal logits: the lower index first); the token is the first index, in the vocabulary's
//   order, at which the running sum of the kept w exceeds u times their sum.
//
// A row belongs to a cluster of up to 8 CTAs that hold its slices in shared memory: the logits are read from memory
// once, whatever the passes, and a few rows still spread over the card.
//
// Weights are integers, exp(.) in units of 2^-42 in 64 bits (2^21 of them sum to less than 2^64): their sums do not depend
// on an order, so that results repeat and all CTAs of a cluster come to the same decisions. They are off by at most 2^-27.9 of
// themselves and half a unit, either way: cut off instead of rounded, and to units of 2^-40, they drew another token in one of
// some hundred rows with a peak and a tail of 10^5 tokens. From fp32 arithmetic the sums of a flat row of 10^5 tokens would
// be off by 10^-4 to 10^-3 of a token, and so would the choice.
//
// The filters keep what lies above a border in (logit, index). It is found without sorting: a histogram over the range that
// holds it, of counts for top_k and of weights for top_p, then over the border's bin alone, whose candidates are listed, until
// that is one logit: bins of equal width in the logit first (even for what a model gives), of equal numbers of floats
// afterwards. The weights' first histogram is kept per part of the row (a warp's share), so that the draw along the row's
// order needs the weights of the border's bin only, and then of the part that the draw falls in.
//
// The weights' arithmetic (about 25 instructions each) and the cluster's barriers bound it, not the logits' bytes (12 us):
// 256 rows of 150001 in bf16 take 39 us for the largest alone, 109 us without a filter, 115 us with top_k 50, 193 us with
// top_p 0.9 (two CTAs per SM hide part of the barriers). One row of 32000: 16 us, a chain of seven barriers. Exponentials
// in fp64 and 64-bit atomics in place of the table and the halves: 584 us for the 193.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "decoder.h"

namespace sb {
namespace k {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 384, kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kMostCtas = 8;            // of a cluster
constexpr int kHeld = 192 * 1024;       // bytes of a slice that fit shared memory
constexpr int kCoarse = 128;            // bins of the first round of weights, per warp
constexpr int kListBytes = 4096;        // of a list of candidates
constexpr int kSettled = 256;           // candidates of a row that are ranked one against another
constexpr int kMostRounds = 6;          // 128 or 256 bins, then at least 128 each of what is left of 2^32 floats
constexpr int kSteps = 64;              // table of 2^(-j / 64)
constexpr int kUnit = 42;               // bits of the largest weight

struct SampleArgs {
  const void* logits;
  int64_t stride;
  const float* uniform;
  SamplingView by;
  int64_t* tokens;
  int vocab, slice;   // slice: of a CTA, in elements
};

template <typename T> __device__ __forceinline__ float value(T x);
template <> __device__ __forceinline__ float value(float x) { return x; }
template <> __device__ __forceinline__ float value(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);   // of values that are T's
template <> __device__ __forceinline__ float narrow(float x) { return x; }
template <> __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
template <typename T> __device__ __forceinline__ T lowest();   // -inf
template <> __device__ __forceinline__ float lowest() { return -INFINITY; }
template <> __device__ __forceinline__ __half lowest() { return __ushort_as_half(0xfc00); }
template <> __device__ __forceinline__ __nv_bfloat16 lowest() { return __ushort_as_bfloat16(0xff80); }

// The largest of a piece, NaN passed over.
template <typename T> __device__ __forceinline__ float largest(uint4 v);
template <> __device__ __forceinline__ float largest<float>(uint4 v) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <> __device__ __forceinline__ float largest<__half>(uint4 v) {
  const __half2* e = reinterpret_cast<const __half2*>(&v);
  const float2 m = __half22float2(__hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3])));
  return fmaxf(m.x, m.y);
}
template <> __device__ __forceinline__ float largest<__nv_bfloat16>(uint4 v) {
  const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&v);
  const float2 m = __bfloat1622float2(__hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3])));
  return fmaxf(m.x, m.y);
}

// Logits as integers of the same order; NaN below all others, the zeros equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// 2^(30 - j / 64), rounded
__constant__ uint32_t kPower[kSteps] = {
    1073741824u, 1062175491u, 1050733751u, 1039415261u, 1028218693u, 1017142735u, 1006186087u, 995347464u,
    984625594u, 974019220u, 963527098u, 953147997u, 942880699u, 932724001u, 922676710u, 912737649u,
    902905651u, 893179563u, 883558244u, 874040567u, 864625413u, 855311680u, 846098274u, 836984114u,
    827968132u, 819049271u, 810226483u, 801498734u, 792865000u, 784324269u, 775875538u, 767517817u,
    759250125u, 751071493u, 742980960u, 734977579u, 727060411u, 719228525u, 711481005u, 703816941u,
    696235434u, 688735596u, 681316545u, 673977412u, 666717336u, 659535466u, 652430958u, 645402981u,
    638450708u, 631573326u, 624770026u, 618040012u, 611382493u, 604796689u, 598281827u, 591837143u,
    585461881u, 579155293u, 572916640u, 566745190u, 560640218u, 554601009u, 548626854u, 542717053u,
};

struct alignas(16) Shared {
  // read by the other CTAs of the cluster; what rounds write anew is there twice and used in turn
  uint32_t low[2][kBins], high[2][kBins];   // halves of the bins' sums
  uint32_t least[2], most[2];               // keys of the candidates
  float top;
  int lowest;
  unsigned long long warp_mass[kWarps];
  uint32_t warp_ties[kWarps];
  // this CTA's own
  uint32_t power[kSteps];                   // 2^(30 - j / 64)
  uint32_t part[3][kWarps][kCoarse];        // sums of each warp's part of the slice, of 16, 16 and 11 bits of the weights
  uint4 list[2][kListBytes / 16];
  int listed[2];
  float rank_value[kSettled];
  unsigned long long rank_weight[kSettled];
  unsigned long long scan[2][kWarps];
  float warp_top[kWarps];
  // what its first warp found out
  unsigned long long all, target, above, before, ties_before, tie;
  double wide_rate;
  float most_of_row, start, start_low, rate, rate_low;
  unsigned long long ties;
  uint32_t lo, border;
  int near, outcome, bin, chosen;
};

constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: sums with it are rounded to integers, in their low bits

static_assert(sizeof(Shared) + kHeld <= 227 * 1024, "a slice beside what a CTA keeps");
// The widest row's sums: all of it in 64 bits, a warp's part of a slice (a slice rounded up to 64, a part to pieces) in words of
// 16, 16 and kUnit - 31 bits of each weight.
constexpr int kMostPart = (kMostVocab / kMostCtas + 64) / kWarps + 2 * 8;
static_assert(kMostVocab <= 1 << (63 - kUnit) && kMostPart <= 1 << 16 && kMostPart <= 1 << (32 - (kUnit - 31)), "sums of weights");

// exp((v - top) / T) in units of 2^-kUnit for v from top down to where it is nothing: 2^-y with y = (top - v) log2(e) / T. With
// k = y rounded to 64ths and g what is left of it, it is 2^(-k / 64) from a table, times 1 - z, z = 1 - 2^-g by three terms of its
// series (the next is 2^-33), in integers: off by up to 2^-27.9 of itself (a quarter each from the table and from z, half from
// the product, which is cut off), where expf would be off by up to 2^-21 and exp in fp64 takes three times as long. g is taken as
// (top log2(e) / T - k / 64) - v log2(e) / T, the former without rounding (top's part is split at 2^-8), the latter and the
// difference with one: top - v would lose what small v have, in 16 bits too (up to 2^-21 of a weight below a top of 10).
__device__ __noinline__ unsigned long long wide_exp(double d, double rate) {   // any finite d and temperature
  return __double2ull_rn(exp(d * rate) * double(1ull << kUnit));
}
constexpr float kNearTop = 65536.f;   // multiples of 2^-8 below it are floats
struct NearWeights {   // temperatures and logits that are floats like others, top log2(e) / T below kNearTop
  float start, start_low;   // top log2(e) / T in multiples of 2^-8, and the rest
  float rate, rate_low;     // log2(e) / T
  const uint32_t* power;
  __device__ __forceinline__ unsigned long long operator()(float v) const {
    const float shifted = fmaf(fmaf(-v, rate, start), float(kSteps), kMagic);
    const uint32_t k = __float_as_uint(shifted);
    const float g = fmaf(-v, rate, fmaf(shifted - kMagic, -1.f / kSteps, start)) + fmaf(-v, rate_low, start_low);
    const float z = g * fmaf(-g, fmaf(-g, 0.0555041087f, 0.240226507f), 0.693147181f);
    const int zi = int(__float_as_uint(fmaf(z, 536870912.f, kMagic)) - 0x4b400000u);   // in units of 2^-29
    const uint32_t p = power[k % kSteps];
    const uint32_t w = p - uint32_t(__mulhi(int(p), zi * 8));
    return (((static_cast<unsigned long long>(w) << (kUnit - 30 + 1)) >> (k / kSteps & 63)) + 1) >> 1;   // rounded
  }
};
struct FarWeights {   // any others
  float top;
  double rate;   // 1 / T
  __device__ __forceinline__ unsigned long long operator()(float v) const {
    return v == top ? 1ull << kUnit : wide_exp(double(v) - double(top), rate);
  }
};

// Bins of equal width in the logit, over a range of floats: 0 holds the largest, n - 1 or n - 2 the least (`start` is a whole
// number, so that the largest comes to lie within half a bin of 0).
struct EvenBins {
  float slope, start;
  __device__ __forceinline__ bool set(float l, float h, int n) {
    const float width = 0.5f * h - 0.5f * l;
    slope = -0.5f * float(n - 2) / width;
    start = fmaf(-slope, h, kMagic);
    return width > 0.f && slope < 0.f && slope > -1e30f && fabsf(slope * h) < 1e6f && fabsf(slope * l) < 1e6f;
  }
  __device__ __forceinline__ int operator()(float v) const { return int(__float_as_uint(fmaf(v, slope, start)) & 0x3ffu); }
};

// Bins of a range of keys, of equal numbers of them: 0 holds the largest.
struct KeyBins {
  uint32_t hi;
  int shift;
  __device__ __forceinline__ void set(uint32_t l, uint32_t h, int n) {
    hi = h;
    shift = max(0, 32 - __clz(h - l) - (31 - __clz(n)));   // (h - l) >> shift is below n, a power of two
  }
  __device__ __forceinline__ int operator()(float v) const { return int((hi - key_of(v)) >> shift); }
};

// a / b rounded up (0 for b = 0): from a quotient of doubles, which is off by little (a division of 64-bit integers takes five
// times as long)
__device__ __forceinline__ unsigned long long quotient(unsigned long long a, unsigned long long b) {
  if (b == 0) return 0;
  unsigned long long q = (unsigned long long)(double(a) / double(b));
  while (q > 0 && q * b >= a) --q;
  while (q * b < a) ++q;
  return q;
}

__device__ __forceinline__ unsigned long long sum_upto(unsigned long long v, int lane) {   // of the lanes up to this one
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long p = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += p;
  }
  return v;
}

template <typename T, bool kHold>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& s = *reinterpret_cast<Shared*>(raw);
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / ctas;

  // ---- the slice, in 16-byte pieces as they lie in memory (the first begins `shift` elements before it), and its largest
  constexpr int kV = 16 / sizeof(T);
  const int begin = min(rank * a.slice, a.vocab), count = min(a.slice, a.vocab - begin);
  const T* from = static_cast<const T*>(a.logits) + row * a.stride + begin;
  const int shift = int(reinterpret_cast<uintptr_t>(from) / sizeof(T) % kV);
  const int pieces = (count + shift + kV - 1) / kV;
  T* held = reinterpret_cast<T*>(raw + sizeof(Shared));   // with -inf before and behind
  auto fetch = [&](int q) {
    alignas(16) T e[kV];
    const int i = q * kV - shift;
    if (i >= 0 && i + kV <= count) return *reinterpret_cast<const uint4*>(from + i);
#pragma unroll
    for (int j = 0; j < kV; ++j) e[j] = i + j >= 0 && i + j < count ? from[i + j] : lowest<T>();
    return *reinterpret_cast<const uint4*>(e);
  };
  auto piece = [&](int q) { return kHold ? reinterpret_cast<const uint4*>(held)[q] : fetch(q); };
  auto at = [&](int i) { return value<T>(kHold ? held[i + shift] : from[i]); };
  // The elements of a piece that are wanted, one by one: a warp goes on with as many as its lanes have at most, not with all
  // that any lane has.
  auto each_of = [&](int q, uint32_t wanted, auto&& f) {
    while (wanted) {
      f(at(q * kV - shift + __ffs(int(wanted)) - 1));
      wanted &= wanted - 1;
    }
  };
  float most = -INFINITY;
#pragma unroll 4
  for (int q = tid; q < pieces; q += kThreads) {
    const uint4 v = fetch(q);
    if (kHold) reinterpret_cast<uint4*>(held)[q] = v;
    most = fmaxf(most, largest<T>(v));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
  if (lane == 0) s.warp_top[warp] = most;
  if (tid < kBins) s.low[0][tid] = s.high[0][tid] = 0;
  if (tid < kSteps) s.power[tid] = kPower[tid];
  if (tid == 0) s.lowest = 0x7fffffff, s.least[0] = ~0u, s.most[0] = 0, s.listed[0] = 0, s.bin = 0, s.above = 0;
  __syncthreads();
  if (warp == 0) {
    most = lane < kWarps ? s.warp_top[lane] : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    if (lane == 0) s.top = most;
  }
  cluster.sync();

  const float temperature = a.by.temperature_of ? a.by.temperature_of[row] : a.by.temperature;
  const float top_p = a.by.top_p_of ? a.by.top_p_of[row] : a.by.top_p;
  const float min_p = a.by.min_p_of ? a.by.min_p_of[row] : a.by.min_p;
  int top_k = a.by.top_k_of ? a.by.top_k_of[row] : a.by.top_k;
  if (top_k <= 0 || top_k > a.vocab) top_k = a.vocab;
  if (warp == 0) {
    most = lane < ctas ? cluster.map_shared_rank(&s, lane)->top : -INFINITY;
#pragma unroll
    for (int d = kMostCtas / 2; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
    if (lane == 0) {
      s.most_of_row = most;
      const double r = 1.0 / double(temperature), l = r * 1.4426950408889634;
      s.wide_rate = r, s.rate = float(l), s.rate_low = float(l - double(float(l)));
      const double at = double(most) * l;
      s.start = float(rint(at * 256.0) / 256.0), s.start_low = float(at - double(s.start));
      s.near = temperature > 1e-20f && temperature < 1e20f && fabs(at) < kNearTop;
      // the least key that counts: weights below are 0 or below min_p
      double cut = -29.9;   // 2^kUnit exp(cut) rounds to 0
      if (min_p > 0.f) cut = fmax(cut, log(double(min_p)));
      const float v = most < INFINITY ? __double2float_ru(double(most) + double(temperature) * fmin(cut, 0.0)) : most;
      s.lo = key_of(fmaxf(v, -3.402823466e38f));
    }
  }
  __syncthreads();
  most = s.most_of_row;

  if (most == -INFINITY) {   // nothing to choose from
    if (rank == 0 && tid == 0) a.tokens[row] = -1;
    cluster.sync();          // the others may still read this CTA's numbers
    return;
  }
  if (!(temperature > 0.f) || top_k == 1 || top_p <= 0.f) {   // the largest, the first of them
    int low = 0x7fffffff;
    for (int q = tid; q < pieces && low == 0x7fffffff; q += kThreads) {
      const uint4 v = piece(q);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = kV - 1; j >= 0; --j)
        if (value<T>(e[j]) == most) low = begin + q * kV - shift + j;
    }
    low = __reduce_min_sync(~0u, low);
    if (lane == 0) atomicMin(&s.lowest, low);
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ctas; ++c) low = min(low, cluster.map_shared_rank(&s, c)->lowest);
      a.tokens[row] = low;
    }
    cluster.sync();
    return;
  }

  const NearWeights near_weight = {s.start, s.start_low, s.rate, s.rate_low, s.power};
  const FarWeights far_weight = {most, s.wide_rate};
  const bool near = s.near;
  auto weight = [&](float v) { return near ? near_weight(v) : far_weight(v); };
  const uint32_t lo = s.lo, hi = key_of(most);

  // ---- the border: kept are keys above it, and the first `ties` of its own
  const int part = (pieces + kWarps - 1) / kWarps;   // of a warp, in pieces
  const int part_begin = warp * part, part_end = min(part_begin + part, pieces);
  constexpr int kListed = kListBytes / int(sizeof(T));
  uint32_t border = lo;
  unsigned long long ties = a.vocab;
  int turn = 0;
  // A first round of weights leaves the parts' sums over its bins: those before `summed` need no second look.
  bool binned = false, coarse_even = false;
  int summed = 0;
  EvenBins coarse;
  KeyBins coarse_keys;
  auto part_sum = [&](int w, int b) {
    return s.part[0][w][b] + (static_cast<unsigned long long>(s.part[1][w][b]) << 16) + (static_cast<unsigned long long>(s.part[2][w][b]) << 32);
  };
  // The candidates that the CTAs have listed (each lane: how many of its CTA, and how many before them): the one at which
  // the sums from the top reach need(their sum), by ranking all against all. Whether there is one.
  auto settle = [&](const bool by_mass, int number, int before, int total, auto&& need_of) {
    float v = 0.f;
    for (int c = 0; c < ctas; ++c) {
      const int i = tid - __shfl_sync(~0u, before, c), n = __shfl_sync(~0u, number, c);
      if (i >= 0 && i < n) v = value<T>(reinterpret_cast<const T*>(cluster.map_shared_rank(&s, c)->list[turn])[i]);
    }
    const unsigned long long own = by_mass && tid < total ? weight(v) : 1ull;
    if (tid < total) s.rank_value[tid] = v, s.rank_weight[tid] = own;
    if (tid == 0) s.outcome = 0;
    __syncthreads();
    unsigned long long all = 0;
    for (int j = lane; j < total; j += 32) all += s.rank_weight[j];
    __syncwarp();
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(~0u, all, d);
    const unsigned long long need = need_of(all);
    if (tid < total) {
      unsigned long long greater = 0, equal = 0;
      for (int j = 0; j < total; ++j) {
        const float x = s.rank_value[j];
        const unsigned long long w = s.rank_weight[j];
        greater += x > v ? w : 0;
        equal += x == v ? w : 0;
      }
      if (greater < need && need <= greater + equal) s.border = key_of(v), s.ties = quotient(need - greater, own), s.outcome = 1;
    }
    __syncthreads();
    turn ^= 1;
    if (s.outcome) border = s.border, ties = s.ties;
    return s.outcome != 0;
  };
  // How many the CTAs have listed, each lane its CTA's; before them; in all, or more than can be settled.
  auto numbers = [&](int& number, int& before) {
    number = lane < ctas ? cluster.map_shared_rank(&s, lane)->listed[turn] : 0;
    int upto = number;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int p = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += p;
    }
    before = upto - number;
    const bool fits = __all_sync(~0u, number <= kListed);
    const int total = __shfl_sync(~0u, upto, 31);
    return fits ? total : kSettled + 1;
  };
  // Finds the key at which the sums from the top reach a target: of counts, or of weights. The ties of a border found
  // before are not summed one by one, but by their number.
  auto descend = [&](const bool by_mass) {
    unsigned long long target = top_k;
    const bool floored = by_mass && ties < (unsigned long long)a.vocab;
    const uint32_t floor = border;
    const unsigned long long floor_weight = floored ? weight(of_key(floor)) : 0, floor_sum = floored ? ties * floor_weight : 0;
    const auto part_of = [&](unsigned long long all) {
      return min(max((unsigned long long)ceil(double(top_p) * double(all + floor_sum)), 1ull), all + floor_sum);
    };
    if (floored && top_k <= kSettled) {   // all that are above the border there is
      const float last = of_key(floor);
      T* to = reinterpret_cast<T*>(s.list[turn]);
      for (int q = tid; q < pieces; q += kThreads) {
        const uint4 p = piece(q);
        const T* e = reinterpret_cast<const T*>(&p);
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < kV; ++j) mine |= uint32_t(value<T>(e[j]) > last) << j;
        if (mine) {
          int i = atomicAdd(&s.listed[turn], __popc(mine));
          each_of(q, mine, [&](float v) { to[i++] = narrow<T>(v); });   // less than top_k
        }
      }
      cluster.sync();
      __syncwarp();
      int number, before;
      const int total = numbers(number, before);
      unsigned long long target = 0, sum = 0;
      if (!settle(true, number, before, total, [&](unsigned long long all) { return sum = all, target = part_of(all); }))
        ties = quotient(target - sum, floor_weight);   // among the border's ties
      return;
    }
    uint32_t low_key = floored ? min(floor + 1, hi) : lo, high_key = hi;   // hi itself where none is above the border
    const bool none = floored && floor >= hi;
    unsigned long long above = 0;
    int list = -1, listed = 0;   // the list that holds the candidates, or the slice does
    for (int round = 0; round < kMostRounds; ++round) {
      EvenBins even;
      KeyBins keys;
      const int bins = round == 0 && by_mass ? kCoarse : kBins;
      const float low = of_key(low_key), high = of_key(high_key);
      const bool by_value = even.set(low, high, bins) && round == 0 && near;
      keys.set(low_key, high_key, bins);
      // a 64-bit sum in two halves: whoever makes the lower one overflow carries
      auto add = [&](uint32_t* lower, uint32_t* upper, unsigned long long w) {
        const uint32_t l = uint32_t(w), old = atomicAdd(lower, l);
        const uint32_t h = uint32_t(w >> 32) + (old + l < old);
        if (h) atomicAdd(upper, h);
      };
      auto add_part = [&](int b, unsigned long long w) {   // without a carry: atomics that return nothing are faster
        atomicAdd(&s.part[0][warp][b], uint32_t(w) & 0xffffu);
        const uint32_t m = uint32_t(w) >> 16, h = uint32_t(w >> 32);
        if (m) atomicAdd(&s.part[1][warp][b], m);
        if (h) atomicAdd(&s.part[2][warp][b], h);
      };
      if (round == 0 && by_mass) {
        for (int i = tid; i < 3 * kWarps * kCoarse; i += kThreads) (&s.part[0][0][0])[i] = 0;
        __syncthreads();
        binned = true, coarse_even = by_value, coarse = even, coarse_keys = keys;
        auto sums = [&](const auto& bin, const auto& weight) {
          for (int q = part_begin + lane; q < part_end; q += 32) {
            const uint4 p = piece(q);
            const T* e = reinterpret_cast<const T*>(&p);
#pragma unroll
            for (int j0 = 0; j0 < kV; j0 += 4) {
              unsigned long long w[4];
              int b[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = weight(value<T>(e[j0 + j])), b[j] = bin(value<T>(e[j0 + j]));
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (value<T>(e[j0 + j]) >= low) add_part(b[j], w[j]);
            }
          }
        };
        auto few = [&] {   // the weights of those that count alone
          for (int q = part_begin + lane; q < part_end; q += 32) {
            const uint4 p = piece(q);
            const T* e = reinterpret_cast<const T*>(&p);
            uint32_t mine = 0;
#pragma unroll
            for (int j = 0; j < kV; ++j) mine |= uint32_t(value<T>(e[j]) >= low) << j;
            each_of(q, mine, [&](float v) { add_part(by_value ? even(v) : keys(v), weight(v)); });
          }
        };
        __syncwarp();
        if (none) {}
        else if (by_value && !floored && !(min_p > 0.f)) sums(even, near_weight);
        else few();
        __syncthreads();
        if (tid < kCoarse) {
          unsigned long long n = 0;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) n += part_sum(w, tid);
          s.low[turn][tid] = uint32_t(n), s.high[turn][tid] = uint32_t(n >> 32);
        }
      } else {
        auto count = [&](float v, const auto& bin) {
          if (!(v >= low && v <= high)) return;
          const int b = bin(v);
          if (by_mass) add(&s.low[turn][b], &s.high[turn][b], weight(v));
          else atomicAdd(&s.low[turn][b], 1u);
        };
        auto counts = [&](const auto& bin) {
          for (int q = tid; q < pieces; q += kThreads) {
            const uint4 p = piece(q);
            const T* e = reinterpret_cast<const T*>(&p);
#pragma unroll
            for (int j = 0; j < kV; ++j) count(value<T>(e[j]), bin);
          }
        };
        if (list >= 0)
          for (int i = tid; i < listed; i += kThreads) count(value<T>(reinterpret_cast<const T*>(s.list[list])[i]), keys);
        else if (by_value) counts(even);
        else counts(keys);
      }
      cluster.sync();
      if (tid < kBins) s.low[turn ^ 1][tid] = s.high[turn ^ 1][tid] = 0;   // all have read it, before this barrier
      if (tid == 0) s.least[turn ^ 1] = ~0u, s.most[turn ^ 1] = 0, s.listed[turn ^ 1] = 0;
      __syncwarp();
      if (warp == 0) {   // neighbouring bins per lane
        unsigned long long n[kBins / 32], sum = 0;
        const int each = bins / 32;
#pragma unroll
        for (int i = 0; i < kBins / 32; ++i) n[i] = 0;
#pragma unroll
        for (int i = 0; i < kBins / 32; i += 4) {
          if (i >= each) break;
          const int at = lane * each + i;
          for (int c0 = 0; c0 < ctas; c0 += 2) {   // loads in flight together
            uint4 l[2], h[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const Shared* o = cluster.map_shared_rank(&s, min(c0 + c, ctas - 1));
              l[c] = *reinterpret_cast<const uint4*>(o->low[turn] + at);
              h[c] = by_mass ? *reinterpret_cast<const uint4*>(o->high[turn] + at) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (c0 + c < ctas) {
                n[i] += l[c].x + (static_cast<unsigned long long>(h[c].x) << 32), n[i + 1] += l[c].y + (static_cast<unsigned long long>(h[c].y) << 32);
                n[i + 2] += l[c].z + (static_cast<unsigned long long>(h[c].z) << 32), n[i + 3] += l[c].w + (static_cast<unsigned long long>(h[c].w) << 32);
              }
          }
        }
#pragma unroll
        for (int i = 0; i < kBins / 32; ++i) sum += n[i];
        const unsigned long long upto = sum_upto(sum, lane), all = __shfl_sync(~0u, upto, 31);
        if (round == 0 && by_mass) target = part_of(all);
        const unsigned long long need = target - above;
        if (lane == 0) s.all = all, s.target = target, s.outcome = round == 0 && (by_mass ? target > all : target >= all);
        if (upto >= need && upto - sum < need) {
          unsigned long long before = upto - sum;
#pragma unroll
          for (int i = 0; i < kBins / 32; ++i)
            if (before < need && before + n[i] >= need) {
              s.bin = lane * each + i, s.above = above + before;
              before = need;   // found
            } else {
              before += n[i];
            }
        }
      }
      __syncthreads();
      target = s.target;
      if (s.outcome) {   // no border among these
        if (by_mass) {   // but among the ties of the one there is
          ties = quotient(target - s.all, floor_weight);
          summed = bins;
        }
        turn ^= 1;
        return;
      }
      above = s.above;
      const int found = s.bin;
      if (round == 0) summed = found;
      // the bin's candidates, and the range of their keys
      const int next = turn;
      uint32_t least = ~0u, greatest = 0;
      auto see = [&](float v) {
        const uint32_t k = key_of(v);
        least = min(least, k), greatest = max(greatest, k);
      };
      T* to = reinterpret_cast<T*>(s.list[next]);
      auto take = [&](const auto& bin) {
        for (int q = tid; q < pieces; q += kThreads) {
          const uint4 p = piece(q);
          const T* e = reinterpret_cast<const T*>(&p);
          uint32_t mine = 0;
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = value<T>(e[j]);
            if (v >= low && v <= high && bin(v) == found) mine |= 1u << j;
          }
          if (mine) {
            int i = atomicAdd(&s.listed[next], __popc(mine));
            each_of(q, mine, [&](float v) {
              see(v);
              if (i < kListed) to[i] = narrow<T>(v);
              ++i;
            });
          }
        }
      };
      if (list >= 0) {
        for (int i = tid; i < listed; i += kThreads) {
          const T e = reinterpret_cast<const T*>(s.list[list])[i];
          const float v = value<T>(e);
          if (v >= low && v <= high && keys(v) == found) see(v), to[atomicAdd(&s.listed[next], 1)] = e;
        }
      } else if (by_value) {
        take(even);
      } else {
        take(keys);
      }
      __syncwarp();
      least = __reduce_min_sync(~0u, least), greatest = __reduce_max_sync(~0u, greatest);
      if (lane == 0 && greatest) atomicMin(&s.least[turn], least), atomicMax(&s.most[turn], greatest);
      cluster.sync();
      __syncwarp();
      if (lane < ctas) {
        const Shared* o = cluster.map_shared_rank(&s, lane);
        least = o->least[turn], greatest = o->most[turn];
      } else {
        least = ~0u, greatest = 0;
      }
      least = __reduce_min_sync(~0u, least), greatest = __reduce_max_sync(~0u, greatest);
      low_key = least, high_key = greatest;
      if (least != greatest) {
        int number, before;
        const int total = numbers(number, before);
        if (total <= kSettled) {
          settle(by_mass, number, before, total, [&](unsigned long long) { return target - above; });
          return;
        }
      }
      listed = s.listed[next];
      list = listed <= kListed ? next : -1;
      turn ^= 1;
      if (least == greatest) break;
    }
    border = low_key;
    if (by_mass) {
      const unsigned long long w = weight(of_key(border));
      ties = w ? quotient(target - above, w) : 0;
    } else {
      ties = target - above;
    }
  };
#pragma unroll 1
  for (int filter = 0; filter < 2; ++filter) {
    __syncwarp();
    if (filter == 0 ? top_k < a.vocab : top_p < 1.f) descend(filter == 1);
  }
  __syncwarp();

  // ---- sums of the kept, per warp's part of the slice
  {
    unsigned long long sum = 0;
    uint32_t equal = 0;
    const float last = of_key(border);
    if (binned) {   // of the bins above the border's, and what of that is above the border
      for (int b = lane; b < summed; b += 32) sum += part_sum(warp, b);
      auto rest = [&](const auto& bin) {
        for (int q = part_begin + lane; q < part_end; q += 32) {
          const uint4 p = piece(q);
          const T* e = reinterpret_cast<const T*>(&p);
          uint32_t mine = 0;
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = value<T>(e[j]);
            equal += v == last;
            mine |= uint32_t(v > last && bin(v) >= summed) << j;
          }
          each_of(q, mine, [&](float v) { sum += weight(v); });
        }
      };
      if (coarse_even) rest(coarse);
      else rest(coarse_keys);
    } else {
      if (border != lo || min_p > 0.f || !near) {   // few (at low temperatures too): their weights alone
        for (int q = part_begin + lane; q < part_end; q += 32) {
          const uint4 p = piece(q);
          const T* e = reinterpret_cast<const T*>(&p);
          uint32_t mine = 0;
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = value<T>(e[j]);
            equal += v == last;
            mine |= uint32_t(v > last) << j;
          }
          each_of(q, mine, [&](float v) { sum += weight(v); });
        }
      } else {
        for (int q = part_begin + lane; q < part_end; q += 32) {
          const uint4 p = piece(q);
          const T* e = reinterpret_cast<const T*>(&p);
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = value<T>(e[j]);
            const unsigned long long w = near_weight(v);
            equal += v == last;
            sum += v > last ? w : 0;
          }
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    equal = __reduce_add_sync(~0u, equal);
    if (lane == 0) s.warp_mass[warp] = sum, s.warp_ties[warp] = equal;
  }
  cluster.sync();
  // The part where the target falls: the sums and ties before it, of all CTAs' parts in order.
  __syncwarp();
  if (warp == 0) {
    const unsigned long long tie = weight(of_key(border));
    constexpr int kParts = kMostCtas * kWarps / 32;
    unsigned long long m[kParts], ahead[kParts], upto[kParts], all = 0, met = 0;
#pragma unroll
    for (int b = 0; b < kParts; ++b) {
      const int j = b * 32 + lane;
      m[b] = 0;
      unsigned long long e = 0;
      if (j < ctas * kWarps) {
        const Shared* o = cluster.map_shared_rank(&s, j / kWarps);
        m[b] = o->warp_mass[j % kWarps], e = o->warp_ties[j % kWarps];
      }
      const unsigned long long es = sum_upto(e, lane);
      ahead[b] = met + es - e;
      m[b] += tie * (ahead[b] < ties ? min(e, ties - ahead[b]) : 0ull);
      met += __shfl_sync(~0u, es, 31);
      upto[b] = all + sum_upto(m[b], lane);
      all = __shfl_sync(~0u, upto[b], 31);
    }
    float u = a.uniform[row];
    u = u > 0.f ? fminf(u, 1.f) : 0.f;   // NaN: 0
    const unsigned long long target = min((unsigned long long)(double(u) * double(all)), all - 1);
    if (lane == 0) s.target = target, s.tie = tie;
#pragma unroll
    for (int b = 0; b < kParts; ++b)
      if (upto[b] > target && upto[b] - m[b] <= target) s.chosen = b * 32 + lane, s.before = upto[b] - m[b], s.ties_before = ahead[b];
  }
  __syncthreads();
  const int chosen = s.chosen;
  const unsigned long long target = s.target, tie = s.tie, before = s.before, ties_before = s.ties_before;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");   // nothing more is read of the others
  if (chosen / kWarps == rank) {   // this CTA's: its threads take the part's neighbouring elements
    const int w = chosen % kWarps;
    const int first = max(0, w * part * kV - shift), end = min(count, (w + 1) * part * kV - shift);
    const int each = (end - first + kThreads - 1) / kThreads;
    const int x = min(first + tid * each, end), y = min(x + each, end);
    unsigned long long equal = 0;
    for (int i = x; i < y; ++i) equal += key_of(at(i)) == border;
    __syncwarp();
    unsigned long long upto = sum_upto(equal, lane);
    if (lane == 31) s.scan[0][warp] = upto;
    __syncthreads();
    unsigned long long seen = ties_before + upto - equal;
    for (int v = 0; v < warp; ++v) seen += s.scan[0][v];
    auto kept = [&](int i, unsigned long long& n) -> unsigned long long {
      const float v = at(i);
      const uint32_t k = key_of(v);
      if (k > border) return weight(v);
      return k == border && n++ < ties ? tie : 0;
    };
    unsigned long long sum = 0, n = seen;
    for (int i = x; i < y; ++i) sum += kept(i, n);
    __syncwarp();
    upto = sum_upto(sum, lane);
    if (lane == 31) s.scan[1][warp] = upto;
    __syncthreads();
    unsigned long long running = before + upto - sum;
    for (int v = 0; v < warp; ++v) running += s.scan[1][v];
    if (running <= target && target < running + sum) {
      n = seen;
      for (int i = x; i < y; ++i) {
        running += kept(i, n);
        if (running > target) {
          a.tokens[row] = begin + i;
          break;
        }
      }
    }
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // nor of this CTA
}

template <typename T, bool kHold>
cudaError_t launch(const SampleArgs& a, int64_t rows, int ctas, size_t smem, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, kHold>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(unsigned(rows * ctas));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {unsigned(ctas), 1, 1};
  c.attrs = at, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, sample_kernel<T, kHold>, a);
}

}  // namespace

cudaError_t sample(const void* logits, int64_t stride, int elem, int64_t rows, int vocab, const float* uniform, const SamplingView& by,
                   int64_t* tokens, int sms, cudaStream_t s) {
  const int size = elem == 1 ? 4 : 2;
  // CTAs per row: slices of at most 128 KB, so that two CTAs mostly share an SM (256 rows of 300 KB: 187 us; 64 KB, three of
  // 256 threads: 209), and more while rows leave half of what the SMs hold idle, with 2048 logits or more each: 37 rows of 32000
  // 23 us, by twice as many CTAs 32, by half as many 26; one row by one CTA 30 us, not 17; 4000 logits by two CTAs 13.2 us, by one
  // 14.5, by four 13.8
  int ctas = 1;
  while (ctas < kMostCtas && (int64_t(vocab) * size > int64_t(ctas) * 128 * 1024 || (rows * ctas * 2 <= sms && vocab > ctas * 2048))) ctas *= 2;
  SampleArgs a = {logits, stride, uniform, by, tokens, vocab, 0};
  a.slice = int((int64_t(vocab) + ctas * 64 - 1) / (ctas * 64) * 64);
  const size_t held = size_t(a.slice) * size + 32;   // and the pieces' overhang
  const bool hold = held <= kHeld;
  const size_t smem = sizeof(Shared) + (hold ? held : 0);
  if (elem == 1) return hold ? launch<float, true>(a, rows, ctas, smem, s) : launch<float, false>(a, rows, ctas, smem, s);
  if (elem == 10) return hold ? launch<__half, true>(a, rows, ctas, smem, s) : launch<__half, false>(a, rows, ctas, smem, s);
  return hold ? launch<__nv_bfloat16, true>(a, rows, ctas, smem, s) : launch<__nv_bfloat16, false>(a, rows, ctas, smem, s);
}

}  // namespace k
}  // namespace sb
