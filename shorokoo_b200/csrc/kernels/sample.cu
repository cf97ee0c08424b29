// The next token of each row of logits, from a given random number:
//   w_i = exp((l_i - max) / T); kept are w_i >= min_p, of these the top_k largest, of these the fewest largest whose sum is
//   at least top_p of theirs (equal logits: the lower index first); the token is the first index, in the vocabulary's
//   order, at which the running sum of the kept w exceeds u times their sum.
//
// The logits' bytes bound it while there are many rows, the chain of passes otherwise. A row belongs to a cluster of
// CTAs that hold its slices in shared memory: the logits are read from memory once, whatever the passes, and a few
// rows still spread over the card.
//
// Weights are integers, 2^40 exp(.) in 64 bits from an exponential in fp64: their sums do not depend on an order, so that
// results repeat and all CTAs of a cluster come to the same decisions, and are off by 2^-41 of the largest weight per
// token. In fp32 the sums would be off by about as much as the gap between neighbours of a flat row.
//
// The filters keep what lies above a border in (logit, index). It is found without sorting: a histogram of 512 bins over
// the range that holds it, of counts for top_k and of weights for top_p, then over the border's bin alone, until that is one
// logit: bins of equal width in the logit first (even for what a model gives), of equal numbers of floats afterwards.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "decoder.h"

namespace sb {
namespace k {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = kThreads;         // one thread merges and scans one bin
constexpr int kMostCtas = 8;            // of a cluster
constexpr int kHeld = 200 * 1024;       // bytes of a slice that fit shared memory
constexpr int kMostRounds = 6;          // 512 bins, then at least 256 each of what is left of 2^32 floats
constexpr double kOne = 1099511627776.0;   // 2^40: the largest weight

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

// Logits as integers of the same order; NaN below all others, the zeros equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Shared {   // each CTA's, read by the others of its cluster
  unsigned long long mass[2][kBins];
  uint32_t count[2][kBins];
  float most, least;
  unsigned long long warp_mass[kWarps];
  uint32_t warp_ties[kWarps];
  // this CTA's own
  unsigned long long scan[kWarps];
  unsigned long long found_above;
  float found[2][kWarps];
  uint32_t range[2];
  int low;
};

// The bins of a range of keys: bin 0 holds the largest.
struct Bins {
  uint32_t lo, hi;
  bool even;      // of equal width in the logit
  float half, scale;
  int shift;
  __device__ __forceinline__ void set(uint32_t l, uint32_t h, bool by_value) {
    lo = l, hi = h;
    half = 0.5f * of_key(h);
    const float width = half - 0.5f * of_key(l);
    scale = float(kBins) / width;
    even = by_value && h - l >= uint32_t(kBins) && width > 0.f && scale < INFINITY && scale > 0.f;
    shift = max(0, 32 - __clz(h - l) - 9);   // (h - l) >> shift is below 512
  }
  __device__ __forceinline__ int bin(uint32_t k, float v) const {
    return even ? min(kBins - 1, int((half - 0.5f * v) * scale)) : int((hi - k) >> shift);
  }
};

template <typename T> struct Slice {
  const T* p;
  int count;
  __device__ __forceinline__ float at(int i) const { return value<T>(p[i]); }
};

template <typename T, bool kHold>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& s = *reinterpret_cast<Shared*>(raw);
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / ctas;

  // ---- the slice, its largest and least logit
  const int begin = min(rank * a.slice, a.vocab);
  Slice<T> z;
  z.count = min(a.slice, a.vocab - begin);
  const T* from = static_cast<const T*>(a.logits) + row * a.stride + begin;
  float most = -INFINITY, least = INFINITY;
  {
    constexpr int kV = 16 / sizeof(T);
    const int shift = int(reinterpret_cast<uintptr_t>(from) / sizeof(T) % kV);   // kept in shared memory: 16-byte copies
    T* held = reinterpret_cast<T*>(raw + (sizeof(Shared) + 15) / 16 * 16);
    z.p = kHold ? held + shift : from;
    auto see = [&](float v) {
      if (v > -INFINITY) most = fmaxf(most, v), least = fminf(least, v);   // not NaN
    };
    const int pieces = (z.count + shift + kV - 1) / kV;
#pragma unroll 4
    for (int q = tid; q < pieces; q += kThreads) {
      const int i = q * kV - shift;
      if (i >= 0 && i + kV <= z.count) {
        const uint4 v = *reinterpret_cast<const uint4*>(from + i);
        if (kHold) *reinterpret_cast<uint4*>(held + q * kV) = v;
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < kV; ++j) see(value<T>(e[j]));
      } else {
        for (int j = max(i, 0); j < min(i + kV, z.count); ++j) {
          if (kHold) held[shift + j] = from[j];
          see(value<T>(from[j]));
        }
      }
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, d)), least = fminf(least, __shfl_xor_sync(~0u, least, d));
  if (lane == 0) s.found[0][warp] = most, s.found[1][warp] = least;
  for (int i = tid; i < kBins; i += kThreads) s.mass[0][i] = 0, s.count[0][i] = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) most = fmaxf(most, s.found[0][w]), least = fminf(least, s.found[1][w]);
    s.most = most, s.least = least, s.low = 0x7fffffff, s.range[0] = s.range[1] = 0;
  }
  cluster.sync();
  most = -INFINITY, least = INFINITY;
  for (int c = 0; c < ctas; ++c) {
    const Shared* o = cluster.map_shared_rank(&s, c);
    most = fmaxf(most, o->most), least = fminf(least, o->least);
  }

  const float temperature = a.by.temperature_of ? a.by.temperature_of[row] : a.by.temperature;
  const float top_p = a.by.top_p_of ? a.by.top_p_of[row] : a.by.top_p;
  const float min_p = a.by.min_p_of ? a.by.min_p_of[row] : a.by.min_p;
  int top_k = a.by.top_k_of ? a.by.top_k_of[row] : a.by.top_k;
  if (top_k <= 0 || top_k > a.vocab) top_k = a.vocab;
  float u = a.uniform[row];
  u = u > 0.f ? fminf(u, 1.f) : 0.f;   // NaN: 0

  if (most == -INFINITY) {   // nothing to choose from
    if (rank == 0 && tid == 0) a.tokens[row] = -1;
    cluster.sync();          // the others may still read this CTA's numbers
    return;
  }
  if (!(temperature > 0.f) || top_k == 1 || top_p <= 0.f) {   // the largest, the first of them
    int low = 0x7fffffff;
    for (int i = tid; i < z.count; i += kThreads)
      if (z.at(i) == most) {
        low = begin + i;
        break;
      }
    low = __reduce_min_sync(~0u, low);
    if (lane == 0) atomicMin(&s.low, low);
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ctas; ++c) low = min(low, cluster.map_shared_rank(&s, c)->low);
      a.tokens[row] = low;
    }
    cluster.sync();
    return;
  }

  // ---- weights
  const double top = most, rate = 1.0 / double(temperature);
  auto weight = [&](float v) -> unsigned long long {
    return v == most ? (unsigned long long)kOne : __double2ull_rn(exp((double(v) - top) * rate) * kOne);
  };
  uint32_t lo;   // the least key that counts: weights below are 0 or below min_p
  {
    double cut = -28.5;   // 2^40 exp(cut) rounds to 0
    if (min_p > 0.f) cut = fmax(cut, log(double(min_p)));
    float v = most < INFINITY ? __double2float_ru(top + double(temperature) * fmin(cut, 0.0)) : most;
    lo = max(key_of(fmaxf(v, -3.402823466e38f)), key_of(least));
  }
  const uint32_t hi = key_of(most);

  // ---- the border: kept are keys above it, and the first `ties` of its own
  uint32_t border = lo;
  unsigned long long ties = a.vocab;
  int buffer = 0;
  // The key at which the sums from the top reach a target; sums of counts, or of weights. `among`: (key, ties) of a border
  // found before, which limits what is summed.
  auto descend = [&](bool by_mass, unsigned long long target) {
    Bins bins;
    bins.set(lo, hi, true);
    unsigned long long above = 0;
    const uint32_t floor = border;
    const unsigned long long floor_sum = by_mass && ties < (unsigned long long)a.vocab ? ties * weight(of_key(floor)) : 0;
    const bool floored = by_mass && ties < (unsigned long long)a.vocab;   // its ties are not summed one by one
    for (int round = 0; round < kMostRounds; ++round) {
      const bool first = round == 0;
      for (int i = tid; i < z.count; i += kThreads) {
        const float v = z.at(i);
        const uint32_t k = key_of(v);
        if (k < bins.lo || k > bins.hi || (floored && k <= floor)) continue;
        const int b = bins.bin(k, v);
        if (by_mass) atomicAdd(&s.mass[buffer][b], weight(v));
        else atomicAdd(&s.count[buffer][b], 1u);
      }
      cluster.sync();
      s.mass[buffer ^ 1][tid] = 0, s.count[buffer ^ 1][tid] = 0;
      unsigned long long n = 0;
      for (int c = 0; c < ctas; ++c) {
        const Shared* o = cluster.map_shared_rank(&s, c);
        n += by_mass ? o->mass[buffer][tid] : o->count[buffer][tid];
      }
      buffer ^= 1;
      unsigned long long upto = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long before = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += before;
      }
      if (lane == 31) s.scan[warp] = upto;
      __syncthreads();
      unsigned long long all = 0, before = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) before = all;
        all += s.scan[w];
      }
      upto += before;
      if (first && by_mass) {
        const double part = double(top_p) * double(all + floor_sum);
        target = min(max((unsigned long long)ceil(part), 1ull), all + floor_sum);
        if (target > all) {   // among the ties of the border there is
          ties = (target - all + weight(of_key(floor)) - 1) / weight(of_key(floor));
          return;
        }
      }
      if (first && !by_mass && target >= all) return;   // all of them
      const unsigned long long need = target - above;
      if (upto >= need && upto - n < need) {
        s.found_above = upto - n;
        // the bin's keys
        uint32_t l, h;
        if (bins.even) {
          auto first_of = [&](int b) {   // the least key whose bin is b or less
            uint32_t x = bins.lo, y = bins.hi;
            while (x < y) {
              const uint32_t m = x + (y - x) / 2;
              if (bins.bin(m, of_key(m)) <= b) y = m;
              else x = m + 1;
            }
            return x;
          };
          l = first_of(tid);
          h = tid == 0 ? bins.hi : first_of(tid - 1) - 1;
        } else {
          h = bins.hi - (uint32_t(tid) << bins.shift);
          const uint32_t reach = (1u << bins.shift) - 1;
          l = h - bins.lo < reach ? bins.lo : h - reach;
        }
        s.range[0] = l, s.range[1] = h;
      }
      __syncthreads();
      above += s.found_above;
      bins.set(s.range[0], s.range[1], false);
      __syncthreads();
      if (bins.lo == bins.hi) break;
    }
    border = bins.lo;
    if (by_mass) {
      const unsigned long long w = weight(of_key(border));
      ties = w ? (target - above + w - 1) / w : 0;
    } else {
      ties = target - above;
    }
  };
  if (top_k < a.vocab) descend(false, top_k);
  if (top_p < 1.f) descend(true, 0);

  // ---- sums of the kept, per warp's part of the slice
  const int part = (a.slice + kWarps - 1) / kWarps;
  const int first = min(warp * part, z.count), end = min(first + part, z.count);
  {
    unsigned long long sum = 0;
    uint32_t equal = 0;
    for (int i = first + lane; i < end; i += 32) {
      const float v = z.at(i);
      const uint32_t k = key_of(v);
      if (k > border) sum += weight(v);
      else if (k == border) ++equal;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    equal = __reduce_add_sync(~0u, equal);
    if (lane == 0) s.warp_mass[warp] = sum, s.warp_ties[warp] = equal;
  }
  cluster.sync();
  // Every warp looks where the target falls; the one whose part it is finds the token.
  const unsigned long long tie = weight(of_key(border));
  unsigned long long all = 0, before = 0, ties_before = 0, mine = 0;
  {
    unsigned long long met = 0;   // ties so far
    for (int j0 = 0; j0 < ctas * kWarps; j0 += 32) {
      const int j = j0 + lane;
      unsigned long long m = 0;
      uint32_t e = 0;
      if (j < ctas * kWarps) {
        const Shared* o = cluster.map_shared_rank(&s, j / kWarps);
        m = o->warp_mass[j % kWarps], e = o->warp_ties[j % kWarps];
      }
      unsigned long long es = e;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long p = __shfl_up_sync(~0u, es, d);
        if (lane >= d) es += p;
      }
      const unsigned long long ahead = met + es - e;
      m += tie * (ahead < ties ? min((unsigned long long)e, ties - ahead) : 0ull);
      unsigned long long ms = m;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long p = __shfl_up_sync(~0u, ms, d);
        if (lane >= d) ms += p;
      }
      const int me = rank * kWarps + warp;
      if (me >= j0 && me < j0 + 32) {
        before = all + __shfl_sync(~0u, ms - m, me - j0);
        mine = __shfl_sync(~0u, m, me - j0);
        ties_before = __shfl_sync(~0u, ahead, me - j0);
      }
      all += __shfl_sync(~0u, ms, 31);
      met += __shfl_sync(~0u, es, 31);
    }
  }
  const unsigned long long target = min((unsigned long long)(double(u) * double(all)), all - 1);
  if (target >= before && target - before < mine) {
    // lanes take neighbouring elements, then all of them those of the lane whose it is
    const int each = (end - first + 31) / 32;
    auto kept = [&](int i, unsigned long long& met) -> unsigned long long {
      const float v = z.at(i);
      const uint32_t k = key_of(v);
      if (k > border) return weight(v);
      if (k == border && met++ < ties) return tie;
      return 0;
    };
    int from = first, to = end, step = each;
    while (true) {
      const int x = min(from + lane * step, to), y = min(x + step, to);
      unsigned long long equal = 0;
      for (int i = x; i < y; ++i) equal += key_of(z.at(i)) == border;
      unsigned long long met = equal;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long p = __shfl_up_sync(~0u, met, d);
        if (lane >= d) met += p;
      }
      met += ties_before - equal;
      const unsigned long long ahead = met;
      unsigned long long sum = 0;
      for (int i = x; i < y; ++i) sum += kept(i, met);
      unsigned long long upto = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long p = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += p;
      }
      upto += before;
      const uint32_t over = __ballot_sync(~0u, upto > target);
      const int l = __ffs(over) - 1;   // there is one: the part's sum reaches beyond the target
      if (step == 1) {
        if (lane == l) a.tokens[row] = begin + x;
        break;
      }
      from = __shfl_sync(~0u, x, l), to = __shfl_sync(~0u, y, l);
      before = __shfl_sync(~0u, upto - sum, l);
      ties_before = __shfl_sync(~0u, ahead, l);
      step = max(1, (to - from + 31) / 32);
    }
  }
  cluster.sync();   // the others may still read this CTA's numbers
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
  // CTAs per row: slices of at most 64 KB, so that several CTAs share an SM, and more while rows leave SMs idle
  int ctas = 1;
  while (ctas < kMostCtas && (int64_t(vocab) * size > int64_t(ctas) * 64 * 1024 || (rows * ctas * 2 <= sms && vocab > ctas * 2048))) ctas *= 2;
  SampleArgs a = {logits, stride, uniform, by, tokens, vocab, 0};
  a.slice = int((int64_t(vocab) + ctas * 64 - 1) / (ctas * 64) * 64);
  const size_t held = size_t(a.slice) * size + 32;
  const bool hold = held <= kHeld;
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (hold ? held : 0);
  if (elem == 1) return hold ? launch<float, true>(a, rows, ctas, smem, s) : launch<float, false>(a, rows, ctas, smem, s);
  if (elem == 10) return hold ? launch<__half, true>(a, rows, ctas, smem, s) : launch<__half, false>(a, rows, ctas, smem, s);
  return hold ? launch<__nv_bfloat16, true>(a, rows, ctas, smem, s) : launch<__nv_bfloat16, false>(a, rows, ctas, smem, s);
}

}  // namespace k
}  // namespace sb
