// The norms around a block's residual, row by row:
//   t = post(x) (or x),   h = residual + scale gate t,   y = norm(h)
// with norm(z) = z w / sqrt(mean(z^2) + eps) + b, or, as a layer norm, of z less its mean.
//
// A row is read once, held in registers in fp32 from its loads to its stores, and written once: memory
// bandwidth bounds many rows, and the chain load, sums, store a single one. y is taken of h before h is
// rounded to its type. The variance of a layer norm is the mean square of differences from the mean, in a
// second sum over the registers: the difference of two large sums would lose it where the mean is large.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "decoder.h"

namespace sb {
namespace k {
namespace {

template <typename T> __device__ __forceinline__ float widen(T x);
template <> __device__ __forceinline__ float widen(float x) { return x; }
template <> __device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow(float x) { return x; }
template <> __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }

// V elements as they lie in memory: 16-byte accesses for V = 8, single elements for V = 1
template <typename T, int V> struct alignas(V == 8 ? 16 : sizeof(T)) Piece { T e[V]; };

template <int V> __device__ __forceinline__ void load_vector(float (&to)[V], const void* p, int64_t at, int elem, float add) {
  if (elem == 1) {
    const Piece<float, V> v = *reinterpret_cast<const Piece<float, V>*>(static_cast<const float*>(p) + at);
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = v.e[e] + add;
  } else if (elem == 10) {
    const Piece<__half, V> v = *reinterpret_cast<const Piece<__half, V>*>(static_cast<const __half*>(p) + at);
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = __half2float(v.e[e]) + add;
  } else {
    const Piece<__nv_bfloat16, V> v = *reinterpret_cast<const Piece<__nv_bfloat16, V>*>(static_cast<const __nv_bfloat16*>(p) + at);
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = __bfloat162float(v.e[e]) + add;
  }
}

// Sums over the threads of a row: a warp, or a whole CTA (`slots`: two sets of 32, used in turn, so that one
// barrier per sum is enough).
template <bool kWarp> struct Row {
  float* slots;
  int turn = 0;
  __device__ __forceinline__ float sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    if (kWarp) return v;
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    float* s = slots + turn * 32;
    turn ^= 1;
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? s[lane] : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
  }
};

// Mean to subtract and factor to multiply by, of the row's values; those past the width are 0.
template <int V, int P, bool kWarp>
__device__ __forceinline__ float2 moments(const float (&z)[P][V], const ResidualNormArgs& a, Row<kWarp>& row, int tid, int stride) {
  float mean = 0.f;
  if (a.layer) {
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) s += z[p][e];
    mean = row.sum(s) * a.per_width;
  }
  float s = 0.f;
#pragma unroll
  for (int p = 0; p < P; ++p)
    if ((tid + p * stride) * V < a.width) {
#pragma unroll
      for (int e = 0; e < V; ++e) s += (z[p][e] - mean) * (z[p][e] - mean);
    }
  return make_float2(mean, rsqrtf(row.sum(s) * a.per_width + a.eps));
}

// P pieces of V elements per thread; S: the type of residual and sum; kMost: threads of a row, at most. 32: a row per
// warp, else per CTA.
template <typename T, typename S, int V, int P, int kMost>
__global__ void __launch_bounds__(kMost == 32 ? 128 : kMost) residual_norm_kernel(const ResidualNormArgs a) {
  constexpr bool kWarp = kMost == 32;
  __shared__ float slots[kWarp ? 1 : 64];
  Row<kWarp> row{slots};
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x, stride = kWarp ? 32 : blockDim.x;
  const int64_t m = kWarp ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (m >= a.rows) return;   // whole warps
  using PT = Piece<T, V>;
  using PS = Piece<S, V>;
  PT x[P], g[P];
  PS r[P];
  float z[P][V];
  const T* xr = static_cast<const T*>(a.x) + m * a.xs;
  const S* rr = static_cast<const S*>(a.residual) + m * a.rs;
  const T* gr = static_cast<const T*>(a.gate) + m * a.gs;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = (tid + p * stride) * V;
    if (at >= a.width) continue;
    x[p] = *reinterpret_cast<const PT*>(xr + at);
    if (a.residual) r[p] = *reinterpret_cast<const PS*>(rr + at);
    if (a.gate) g[p] = *reinterpret_cast<const PT*>(gr + at);
  }
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < V; ++e) z[p][e] = (tid + p * stride) * V < a.width ? widen<T>(x[p].e[e]) : 0.f;
  if (a.post_weight) {
    const float2 c = moments<V, P, kWarp>(z, a, row, tid, stride);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int at = (tid + p * stride) * V;
      if (at >= a.width) continue;
      float w[V], b[V];
      load_vector<V>(w, a.post_weight, at, a.weight_elem, a.offset);
      if (a.post_bias) load_vector<V>(b, a.post_bias, at, a.weight_elem, 0.f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        z[p][e] = (z[p][e] - c.x) * c.y * w[e];
        if (a.post_bias) z[p][e] += b[e];
      }
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = (tid + p * stride) * V;
    if (at >= a.width) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v = z[p][e] * a.scale;
      if (a.gate) v *= widen<T>(g[p].e[e]);
      z[p][e] = a.residual ? widen<S>(r[p].e[e]) + v : v;
    }
    if (a.sum) {
      PS h;
#pragma unroll
      for (int e = 0; e < V; ++e) h.e[e] = narrow<S>(z[p][e]);
      *reinterpret_cast<PS*>(static_cast<S*>(a.sum) + m * a.ss + at) = h;
    }
  }
  if (!a.y) return;
  const float2 c = moments<V, P, kWarp>(z, a, row, tid, stride);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = (tid + p * stride) * V;
    if (at >= a.width) continue;
    float w[V], b[V];
    load_vector<V>(w, a.weight, at, a.weight_elem, a.offset);
    if (a.bias) load_vector<V>(b, a.bias, at, a.weight_elem, 0.f);
    PT y;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float v = (z[p][e] - c.x) * c.y * w[e];
      y.e[e] = narrow<T>(a.bias ? v + b[e] : v);
    }
    *reinterpret_cast<PT*>(static_cast<T*>(a.y) + m * a.ys + at) = y;
  }
}

template <typename T, typename S, int V, int P>
void start(const ResidualNormArgs& a, int threads, cudaStream_t s) {
  if (threads == 32) {
    constexpr int kRows = 4;   // of a CTA
    residual_norm_kernel<T, S, V, P, 32><<<unsigned((a.rows + kRows - 1) / kRows), 32 * kRows, 0, s>>>(a);
  } else if (threads <= 256) {
    residual_norm_kernel<T, S, V, P, 256><<<unsigned(a.rows), threads, 0, s>>>(a);
  } else {
    residual_norm_kernel<T, S, V, P, 1024><<<unsigned(a.rows), threads, 0, s>>>(a);
  }
}

template <typename T, typename S>
cudaError_t launch(const ResidualNormArgs& a, bool wide, int sms, cudaStream_t s) {
  const int v = wide ? 8 : 1;
  const int pieces = (a.width + v - 1) / v;
  // Pieces per thread: with rows for every SM, four 16-byte pieces (or 16 elements), so that a row takes few
  // warps; otherwise one (four), so that it takes many.
  const bool many = a.rows >= 2 * int64_t(sms);
  int each = wide ? (many ? 4 : 1) : (many ? 16 : 4);
  const int most = wide ? 4 : 32;
  while (each < most && pieces > 1024 * each) each *= 2;
  int threads = 32;
  while (threads < 1024 && threads * each < pieces) threads *= 2;
  if (wide) {
    if (each == 1) start<T, S, 8, 1>(a, threads, s);
    else if (each == 2) start<T, S, 8, 2>(a, threads, s);
    else start<T, S, 8, 4>(a, threads, s);
  } else {
    if (each == 4) start<T, S, 1, 4>(a, threads, s);
    else if (each <= 16) start<T, S, 1, 16>(a, threads, s);
    else start<T, S, 1, 32>(a, threads, s);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t residual_norm(const ResidualNormArgs& args, int elem, int sum_elem, int sms, cudaStream_t s) {
  ResidualNormArgs a = args;
  a.per_width = 1.f / float(a.width);
  // 16-byte pieces: 8 elements, of each row, of whatever type
  auto fits = [&](const void* p, int64_t stride) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride % 8 == 0 || a.rows == 1));
  };
  const bool wide = a.width % 8 == 0 && fits(a.x, a.xs) && fits(a.residual, a.rs) && fits(a.sum, a.ss) &&
                    fits(a.y, a.ys) && fits(a.gate, a.gs) && fits(a.weight, 0) && fits(a.bias, 0) &&
                    fits(a.post_weight, 0) && fits(a.post_bias, 0);
  if (elem == 1) return launch<float, float>(a, wide, sms, s);
  if (elem == 10) return sum_elem == 1 ? launch<__half, float>(a, wide, sms, s) : launch<__half, __half>(a, wide, sms, s);
  return sum_elem == 1 ? launch<__nv_bfloat16, float>(a, wide, sms, s) : launch<__nv_bfloat16, __nv_bfloat16>(a, wide, sms, s);
}

}  // namespace k
}  // namespace sb
