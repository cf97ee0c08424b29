// The norms around a block's residual, row by row:
//   t = post(x) (or x),   h = residual + scale gate t,   y = norm(h)
// with norm(z) = z w / sqrt(mean(z^2) + eps) + b, or, as a layer norm, of z less its mean.
//
// A row is read once, held in registers in fp32 from its loads to its stores, and written once: memory bandwidth bounds many
// rows, and the chain load, sums, store a single one. y is taken of h before h is rounded to its type. The variance of a
// layer norm is the mean square of differences from the mean, in a second sum over the registers: the difference of two
// large sums would lose it where the mean is large.
// Rows of more than 16384 elements take 32 to 40 registers of each of 1024 threads for their values, of which a part spills:
// 800 rows of 17000 in bf16 with both norms 51 us, of 16000 38; 400 rows of 32768 45 us, of 32767 80. (With edges, the
// streaming form for up to 256 threads spills 64 to 76 bytes a thread, too.)
//
// Measured: 12608 rows of 768 in fp32 36 us (5.4 TB/s, 0.83 of the measured rate); 4099 of 4096 in bf16 with both norms
// and a gate 39 us (3.5 TB/s: 840 instructions per warp and row bound it); one row of 4096 replayed 4.3 us.
//
// Threads take pieces of 8 elements that begin where memory has 16-byte boundaries: with a row that begins s elements
// behind one, the first piece has s elements before the row, which count as none. Rows of an odd width so come in wide
// accesses too (777 of 11001 in fp16 with a residual in fp32: 53 us, element by element 95); only the weights, which lie
// otherwise, are shifted into place. Tensors whose rows begin unlike each other, and weights that are not 16-byte aligned, go
// element by element (4099 rows of 4096 in bf16 with a residual 95 us, not 28).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

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

// Words of two 16-bit elements or one of 32 bits
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t w);
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack(float x, float y);
template <> __device__ __forceinline__ uint32_t pack<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// V elements as they lie in memory: 16-byte accesses for V = 8, single elements for V = 1
template <typename T, int V> struct alignas(V == 8 ? 16 : sizeof(T)) Piece {
  T e[V];
  __device__ __forceinline__ void widened(float (&z)[V]) const {
    if constexpr (V == 8 && sizeof(T) == 2) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack<T>(w[i]);
        z[2 * i] = f.x, z[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = widen<T>(e[i]);
    }
  }
  __device__ __forceinline__ void narrowed(const float (&z)[V]) {
    if constexpr (V == 8 && sizeof(T) == 2) {
      uint32_t* w = reinterpret_cast<uint32_t*>(e);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack<T>(z[2 * i], z[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = narrow<T>(z[i]);
    }
  }
};

// Which of a piece's elements are in the row: `at` is the index of its first, below the width. Without edges, pieces
// begin with the row and the width is a whole number of them.
template <int V, bool kEdges> __device__ __forceinline__ bool whole(int at, int width) { return V == 1 || !kEdges || (at >= 0 && at + V <= width); }
__device__ __forceinline__ bool inside(int i, int width) { return i >= 0 && i < width; }

// (Not inline: code that only a row's first and last piece run, at every access.)
template <typename T> __device__ __noinline__ Piece<T, 8> load_part(const T* row, int at, int width) {
  Piece<T, 8> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v.e[e] = inside(at + e, width) ? row[at + e] : narrow<T>(0.f);
  return v;
}
template <typename T> __device__ __noinline__ void store_part(T* row, int at, int width, Piece<T, 8> v) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (inside(at + e, width)) row[at + e] = v.e[e];
}
template <typename T, int V, bool kEdges> __device__ __forceinline__ Piece<T, V> load(const T* row, int at, int width) {
  if constexpr (V == 8 && kEdges)
    if (!whole<V, kEdges>(at, width)) return load_part<T>(row, at, width);
  return *reinterpret_cast<const Piece<T, V>*>(row + at);
}
template <typename T, int V, bool kEdges> __device__ __forceinline__ void store(T* row, int at, int width, const float (&z)[V]) {
  Piece<T, V> v;
  v.narrowed(z);
  if constexpr (V == 8 && kEdges)
    if (!whole<V, kEdges>(at, width)) return store_part<T>(row, at, width, v);
  *reinterpret_cast<Piece<T, V>*>(row + at) = v;
}

// A piece of weights, which are aligned as a whole, from any element: `skip` elements into the 16 from the boundary
// before it. (Read-only loads: they need not wait for the stores before them.)
template <typename W, bool kStaged> __device__ __forceinline__ Piece<W, 8> shifted(const W* p, int skip) {
  Piece<W, 8> v;
  uint32_t* w = reinterpret_cast<uint32_t*>(v.e);
  auto words = [](uint32_t* to, const W* from, int n) {
#pragma unroll
    for (int i = 0; i < n; i += 4) {
      const uint4* at = reinterpret_cast<const uint4*>(from) + i / 4;
      const uint4 q = kStaged ? *at : __ldg(at);
      to[i] = q.x, to[i + 1] = q.y, to[i + 2] = q.z, to[i + 3] = q.w;
    }
  };
  if constexpr (sizeof(W) == 4) {
    if (skip % 4 == 0) {
      words(w, p, 8);
    } else {
      uint32_t x[12];
      words(x, p - skip % 4, 12);
#pragma unroll
      for (int e = 0; e < 10; ++e) x[e] = skip & 2 ? x[e + 2] : x[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = skip & 1 ? x[e + 1] : x[e];
    }
  } else {
    if (skip == 0) {
      words(w, p, 4);
    } else {
      uint32_t x[8];
      words(x, p - skip, 8);
#pragma unroll
      for (int i = 0; i < 6; ++i) x[i] = skip & 4 ? x[i + 2] : x[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) x[i] = skip & 2 ? x[i + 1] : x[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(x[i], x[i + 1], (skip & 1) * 16);
    }
  }
  return v;
}
// kStaged: from a copy in shared memory, laid out as the rows' pieces are, with zeros before and behind.
constexpr int kPad = 16;   // of them, at least, on either side
template <typename W, int V, bool kEdges, bool kStaged>
__device__ __forceinline__ void weights(float (&to)[V], const void* p, int at, int width) {
  const W* w = static_cast<const W*>(p);
  if constexpr (kStaged) {
    shifted<W, true>(w + at, 0).widened(to);
  } else if constexpr (V == 1) {
    to[0] = widen<W>(__ldg(w + at));
  } else if constexpr (!kEdges) {
    shifted<W, false>(w + at, 0).widened(to);
  } else {
    const int skip = at & 7;
    if (at >= skip && at + (skip ? 16 - skip : 8) <= width) shifted<W, false>(w + at, skip).widened(to);
    else load_part<W>(w, at, width).widened(to);
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

// Mean to subtract and factor to multiply by, of the row's values; those outside it are 0.
template <int V, int P, bool kEdges, bool kWarp>
__device__ __forceinline__ float2 moments(const float (&z)[P][V], const ResidualNormArgs& a, Row<kWarp>& row, int first, int stride) {
  float mean = 0.f, s = 0.f;
  if (a.layer) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) s += z[p][e];
    // The product with the rounded 1 / width, and what that leaves of the sum: without the latter equal values would be off
    // their mean, by as much as a row's spread may be. (A division there: 777 rows of 11001 55 us, not 54.)
    s = row.sum(s);
    mean = s * a.per_width;
    mean = fmaf(fmaf(-mean, float(a.width), s), a.per_width, mean);
    s = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int at = first + p * stride;
      if (at >= a.width) continue;
      if (whole<V, kEdges>(at, a.width)) {
#pragma unroll
        for (int e = 0; e < V; ++e) s += (z[p][e] - mean) * (z[p][e] - mean);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (inside(at + e, a.width)) s += (z[p][e] - mean) * (z[p][e] - mean);
      }
    }
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) s += z[p][e] * z[p][e];
  }
  return make_float2(mean, rsqrtf(row.sum(s) * a.per_width + a.eps));
}

// z becomes (z - mean) factor w + b; elements outside the row stay 0.
template <typename W, int V, int P, bool kEdges, bool kStaged>
__device__ __forceinline__ void apply(float (&z)[P][V], float2 c, const void* w, const void* b, const ResidualNormArgs& a, int first, int stride) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = first + p * stride;
    if (at >= a.width) continue;
    float f[V], g[V];
    weights<W, V, kEdges, kStaged>(f, w, at, a.width);
    if (b) weights<W, V, kEdges, kStaged>(g, b, at, a.width);
    if (a.layer) {
#pragma unroll
      for (int e = 0; e < V; ++e) z[p][e] -= c.x;
    }
    if (a.offset != 0.f) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = whole<V, kEdges>(at, a.width) || inside(at + e, a.width) ? f[e] + a.offset : 0.f;
    }
    if (b) {
#pragma unroll
      for (int e = 0; e < V; ++e) z[p][e] = fmaf(z[p][e] * c.y, f[e], g[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) z[p][e] = z[p][e] * c.y * f[e];
    }
  }
}

struct Vectors {   // the arguments' or copies of them
  const void *weight, *bias, *post_weight, *post_bias, *gate;
};

// A row from its x in z on; residual and gate come by r(p, at) and g(p, at).
template <typename T, typename S, typename W, int V, int P, bool kEdges, bool kStaged, bool kWarp, typename R, typename G>
__device__ __forceinline__ void finish(float (&z)[P][V], const ResidualNormArgs& a, const Vectors& w, int64_t m, Row<kWarp>& row, int first,
                                       int stride, R&& r, G&& g) {
  if (a.post_weight) apply<W, V, P, kEdges, kStaged>(z, moments<V, P, kEdges, kWarp>(z, a, row, first, stride), w.post_weight, w.post_bias, a, first, stride);
  S* sum = static_cast<S*>(a.sum) + m * a.ss;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = first + p * stride;
    if (at >= a.width) continue;
    if (a.scale != 1.f) {
#pragma unroll
      for (int e = 0; e < V; ++e) z[p][e] *= a.scale;
    }
    float f[V];
    if (a.gate) {
      if (a.gs == 0) weights<T, V, kEdges, kStaged>(f, w.gate, at, a.width);
      else g(p, at).widened(f);
#pragma unroll
      for (int e = 0; e < V; ++e) z[p][e] *= f[e];
    }
    if (a.residual) {
      r(p, at).widened(f);
#pragma unroll
      for (int e = 0; e < V; ++e) z[p][e] += f[e];
    }
    if (!whole<V, kEdges>(at, a.width)) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!inside(at + e, a.width)) z[p][e] = 0.f;
    }
    if (a.sum) store<S, V, kEdges>(sum, at, a.width, z[p]);
  }
  if (!a.y) return;
  apply<W, V, P, kEdges, kStaged>(z, moments<V, P, kEdges, kWarp>(z, a, row, first, stride), w.weight, w.bias, a, first, stride);
  T* y = static_cast<T*>(a.y) + m * a.ys;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int at = first + p * stride;
    if (at < a.width) store<T, V, kEdges>(y, at, a.width, z[p]);
  }
}

// Elements of row m before its first 16-byte boundary: -at of the first piece.
template <typename T, bool kEdges> __device__ __forceinline__ int overhang(const ResidualNormArgs& a, int64_t m) {
  constexpr int kEach = 16 / sizeof(T);
  return !kEdges ? 0 : int(reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + m * a.xs) / sizeof(T) % kEach);
}

// Few rows, or short ones. P pieces of V elements per thread; S: the type of residual and sum; W: of the weights; kMost:
// threads of a row, at most. 32: a row per warp, else per CTA.
template <typename T, typename S, typename W, int V, int P, bool kEdges, int kMost>
__global__ void __launch_bounds__(kMost == 32 ? 128 : kMost) residual_norm_kernel(const ResidualNormArgs a) {
  constexpr bool kWarp = kMost == 32;
  __shared__ float slots[kWarp ? 1 : 64];
  Row<kWarp> row{slots};
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x, stride = (kWarp ? 32 : blockDim.x) * V;
  const int64_t m = kWarp ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (m >= a.rows) return;   // whole warps
  const int first = tid * V - overhang<T, kEdges>(a, m);
  Piece<T, V> g[P];
  Piece<S, V> r[P];
  float z[P][V];
  {
    Piece<T, V> x[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int at = first + p * stride;
      if (at >= a.width) continue;
      x[p] = load<T, V, kEdges>(static_cast<const T*>(a.x) + m * a.xs, at, a.width);
      if (a.residual) r[p] = load<S, V, kEdges>(static_cast<const S*>(a.residual) + m * a.rs, at, a.width);
      if (a.gate && a.gs != 0) g[p] = load<T, V, kEdges>(static_cast<const T*>(a.gate) + m * a.gs, at, a.width);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (first + p * stride < a.width) {
        x[p].widened(z[p]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) z[p][e] = 0.f;
      }
    }
  }
  const Vectors w = {a.weight, a.bias, a.post_weight, a.post_bias, a.gate};
  finish<T, S, W, V, P, kEdges, false, kWarp>(z, a, w, m, row, first, stride, [&](int p, int) { return r[p]; }, [&](int p, int) { return g[p]; });
}

// Many rows: CTAs that stay and take every gridDim.x-th row, whose inputs arrive in shared memory (cp.async, a ring of
// rows) while the rows before are computed. A row comes as the 16-byte pieces of memory that it lies in (the bytes before
// it in the first piece are of the same allocation, those behind it are not read).
__device__ __forceinline__ void copy_row(uint8_t* to, const uint8_t* from, int bytes, int tid, int threads) {
  const int head = int(reinterpret_cast<uintptr_t>(from) % 16);
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  for (int q = tid * 16; q < head + bytes; q += threads * 16) {
    const int n = min(16, head + bytes - q);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + q), "l"(from - head + q), "r"(n) : "memory");
  }
}

struct RowRing {
  int stages, r, g, bytes;   // offsets of residual and gate in a stage, and a stage's bytes
  int vectors;               // with edges: where the copies of the weights begin
};

template <typename T, typename S, typename W, int P, bool kEdges, int kMost, int kCtas>
__global__ void __launch_bounds__(kMost, kCtas) residual_norm_stream(const ResidualNormArgs a, const RowRing ring) {
  constexpr int V = 8;
  extern __shared__ __align__(16) uint8_t held[];
  __shared__ float slots[64];
  Row<false> row{slots};
  const int tid = threadIdx.x, stride = blockDim.x * V;
  const bool gates = a.gate && a.gs != 0;   // rows of them
  auto row_of = [](const void* p, int64_t m, int64_t s, int size) { return static_cast<const uint8_t*>(p) + m * s * size; };
  auto copy = [&](int64_t m, int stage) {
    if (m < a.rows) {
      uint8_t* to = held + stage * ring.bytes;
      copy_row(to, row_of(a.x, m, a.xs, sizeof(T)), a.width * int(sizeof(T)), tid, blockDim.x);
      if (a.residual) copy_row(to + ring.r, row_of(a.residual, m, a.rs, sizeof(S)), a.width * int(sizeof(S)), tid, blockDim.x);
      if (gates) copy_row(to + ring.g, row_of(a.gate, m, a.gs, sizeof(T)), a.width * int(sizeof(T)), tid, blockDim.x);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Vectors w = {a.weight, a.bias, a.post_weight, a.post_bias, a.gs == 0 ? a.gate : nullptr};
  if constexpr (kEdges) {   // all rows of a CTA begin alike: gridDim.x is a multiple of 8
    uint8_t* to = held + ring.vectors;
    const int before = kPad + overhang<T, kEdges>(a, blockIdx.x);
    auto stage = [&](const void*& p, auto one) {
      using E = decltype(one);
      if (p == nullptr) return;
      E* v = reinterpret_cast<E*>(to);
      for (int i = tid; i < a.width + 3 * kPad; i += blockDim.x)
        v[i] = inside(i - before, a.width) ? static_cast<const E*>(p)[i - before] : narrow<E>(0.f);
      p = v + before;
      to += ((a.width + 3 * kPad) * int(sizeof(E)) + 15) / 16 * 16;
    };
    stage(w.weight, W()), stage(w.bias, W()), stage(w.post_weight, W()), stage(w.post_bias, W()), stage(w.gate, T());
  }
  for (int i = 0; i < ring.stages - 1; ++i) copy(blockIdx.x + int64_t(i) * gridDim.x, i);
  int in = ring.stages - 1, out = 0;
  for (int64_t m = blockIdx.x; m < a.rows; m += gridDim.x) {
    if (ring.stages == 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (ring.stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
    __syncthreads();   // the row is there, and the one before it done with
    copy(m + int64_t(ring.stages - 1) * gridDim.x, in);
    in = in + 1 == ring.stages ? 0 : in + 1;
    const uint8_t* from = held + out * ring.bytes;
    out = out + 1 == ring.stages ? 0 : out + 1;
    auto begin = [](const uint8_t* p) { return int(reinterpret_cast<uintptr_t>(p) % 16); };
    const T* x = reinterpret_cast<const T*>(from + begin(row_of(a.x, m, a.xs, sizeof(T))));
    const S* r = reinterpret_cast<const S*>(from + ring.r + begin(row_of(a.residual, m, a.rs, sizeof(S))));
    const T* g = reinterpret_cast<const T*>(from + ring.g + begin(row_of(a.gate, m, a.gs, sizeof(T))));
    const int first = tid * V - overhang<T, kEdges>(a, m);
    float z[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int at = first + p * stride;
      if (at < a.width) {
        load<T, V, false>(x, at, a.width).widened(z[p]);
        if (!whole<V, kEdges>(at, a.width)) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (!inside(at + e, a.width)) z[p][e] = 0.f;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) z[p][e] = 0.f;
      }
    }
    finish<T, S, W, V, P, kEdges, kEdges, false>(z, a, w, m, row, first, stride, [&](int, int at) { return load<S, V, false>(r, at, a.width); },
                                                 [&](int, int at) { return load<T, V, false>(g, at, a.width); });
  }
}

template <typename T, typename S, typename W, int P, bool kEdges, int kMost, int kCtas>
cudaError_t stream(const ResidualNormArgs& a, RowRing ring, size_t smem, int threads, int ctas, int sms, cudaStream_t s) {
  const auto kernel = residual_norm_stream<T, S, W, P, kEdges, kMost, kCtas>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
  if (e != cudaSuccess) return e;
  int64_t grid = std::min<int64_t>(a.rows, int64_t(ctas) * sms);
  if (kEdges && grid >= 8) grid -= grid % 8;
  kernel<<<unsigned(grid), threads, smem, s>>>(a, ring);
  return cudaGetLastError();
}

// kLong: rows that take all of 1024 threads
template <typename T, typename S, typename W, int V, int P, bool kEdges, bool kLong = false>
cudaError_t start(const ResidualNormArgs& a, int threads, cudaStream_t s) {
  if constexpr (kLong) {
    residual_norm_kernel<T, S, W, V, P, kEdges, 1024><<<unsigned(a.rows), 1024, 0, s>>>(a);
  } else if (threads == 32) {
    constexpr int kRows = 4;   // of a CTA
    residual_norm_kernel<T, S, W, V, P, kEdges, 32><<<unsigned((a.rows + kRows - 1) / kRows), 32 * kRows, 0, s>>>(a);
  } else if (threads <= 256) {
    residual_norm_kernel<T, S, W, V, P, kEdges, 256><<<unsigned(a.rows), threads, 0, s>>>(a);
  } else {
    residual_norm_kernel<T, S, W, V, P, kEdges, 1024><<<unsigned(a.rows), threads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

// Pieces of 8 elements, or single ones where rows begin unlike each other.
template <typename T, typename S, typename W, bool kEdges>
cudaError_t launch_wide(const ResidualNormArgs& a, int sms, cudaStream_t s) {
  const int pieces = (a.width + 7) / 8 + (kEdges ? 1 : 0);
  // Many rows of 1024 elements or more: two pieces per thread (4099 rows of 4096 in bf16 with both norms and a gate: 39 us,
  // one piece 45, four 46; without the ring 97). Shorter rows go a warp each without it (12608 of 768 in fp32: 36 us, 39 with;
  // 12000 of 768 in bf16 with both norms 25 and 29, of 1280 45 and 41). Many: enough for every CTA (1200 of 4096 16 us, 21
  // without), with edges, whose weights have to be staged first, for every CTA to take two (900 of 4099 26 us without, 32 with).
  constexpr int kEach = 2;
  RowRing ring;
  const int pad = kEdges ? 48 : 0;   // a row that begins and ends inside a piece: what such pieces hold besides
  auto up = [](int n) { return (n + 15) / 16 * 16; };
  ring.r = up(a.width * int(sizeof(T))) + pad;
  ring.g = ring.r + (a.residual ? up(a.width * int(sizeof(S))) + pad : 0);
  ring.bytes = ring.g + (a.gate && a.gs != 0 ? up(a.width * int(sizeof(T))) + pad : 0);
  int threads = std::max(64, (pieces + 32 * kEach - 1) / (32 * kEach) * 32);
  const int room = 216 * 1024;
  int staged = 0;   // copies of the weights
  if (kEdges) {
    for (const void* p : {a.weight, a.bias, a.post_weight, a.post_bias})
      if (p) staged += up((a.width + 3 * kPad) * int(sizeof(W)));
    if (a.gate && a.gs == 0) staged += up((a.width + 3 * kPad) * int(sizeof(T)));
  }
  const int ctas = std::min(threads <= 256 ? 1280 / threads : 1024 / threads, room / (2 * ring.bytes + staged));
  if (ctas == 1) threads = 1024;   // one row at a time: more warps hide more of its chain (777 of 11001: 53 us, 704 threads 59)
  if (pieces >= 128 && threads <= 1024 && ctas > 0 && a.rows >= (kEdges ? 2 : 1) * int64_t(ctas) * sms && int64_t(ctas) * sms >= 8) {
    ring.stages = std::min(4, (room / ctas - staged) / ring.bytes);
    ring.vectors = ring.stages * ring.bytes;
    const size_t smem = size_t(ring.vectors) + staged;
    if (threads <= 256) return stream<T, S, W, kEach, kEdges, 256, 5>(a, ring, smem, threads, ctas, sms, s);
    return stream<T, S, W, kEach, kEdges, 1024, 1>(a, ring, smem, threads, ctas, sms, s);
  }
  // Pieces per thread: with rows for every SM four, so that a row takes few warps; otherwise one, so that it takes many.
  int each = a.rows >= 2 * int64_t(sms) || pieces > 1024 ? 4 : 1;
  threads = 32;
  while (threads < 1024 && threads * each < pieces) threads *= 2;
  if (each == 1) return start<T, S, W, 8, 1, kEdges>(a, threads, s);
  if constexpr (kEdges)
    if (pieces > 4096) return start<T, S, W, 8, 5, kEdges, true>(a, threads, s);   // 32768 elements and an overhang
  return start<T, S, W, 8, 4, kEdges>(a, threads, s);
}

template <typename T, typename S, typename W>
cudaError_t launch_single(const ResidualNormArgs& a, int sms, cudaStream_t s) {
  const int each = a.width > 16384 ? 32 : a.rows >= 2 * int64_t(sms) || a.width > 4096 ? 16 : 4;
  int threads = 32;
  while (threads < 1024 && threads * each < a.width) threads *= 2;
  if (each == 4) return start<T, S, W, 1, 4, false>(a, threads, s);
  if (each == 16) return start<T, S, W, 1, 16, false>(a, threads, s);
  return start<T, S, W, 1, 32, false, true>(a, threads, s);
}

enum Form { kSingle, kPieces, kWithEdges };
template <typename T, typename S, typename W>
cudaError_t launch_form(const ResidualNormArgs& a, Form form, int sms, cudaStream_t s) {
  if (form == kPieces) return launch_wide<T, S, W, false>(a, sms, s);
  return form == kWithEdges ? launch_wide<T, S, W, true>(a, sms, s) : launch_single<T, S, W>(a, sms, s);
}
template <typename T, typename S>
cudaError_t launch(const ResidualNormArgs& a, Form form, int sms, cudaStream_t s) {
  return a.weight_elem == 1 ? launch_form<T, S, float>(a, form, sms, s) : launch_form<T, S, T>(a, form, sms, s);
}

}  // namespace

cudaError_t residual_norm(const ResidualNormArgs& args, int elem, int sum_elem, int sms, cudaStream_t s) {
  ResidualNormArgs a = args;
  a.per_width = 1.f / float(a.width);
  // Rows begin alike, in elements from a 16-byte boundary: 8 elements apart for the 16-bit types, 4 for 32-bit ones.
  const int per = elem == 1 ? 4 : 8, sum_per = sum_elem == 1 ? 4 : 8;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(a.x) / (16 / per);
  auto alike = [&](const void* p, int64_t stride, int n) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) / (16 / n) - begin) % n == 0 && (a.rows == 1 || (stride - a.xs) % n == 0));
  };
  auto whole = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool wide = alike(a.residual, a.rs, sum_per) && alike(a.sum, a.ss, sum_per) && alike(a.y, a.ys, per) &&
                    (a.gs == 0 ? whole(a.gate) : alike(a.gate, a.gs, per)) && whole(a.weight) && whole(a.bias) && whole(a.post_weight) &&
                    whole(a.post_bias);
  const bool edges = a.width % 8 != 0 || begin % per != 0 || (a.rows > 1 && a.xs % per != 0);
  const Form form = !wide ? kSingle : edges ? kWithEdges : kPieces;
  if (elem == 1) return launch_form<float, float, float>(a, form, sms, s);
  if (elem == 10) return sum_elem == 1 ? launch<__half, float>(a, form, sms, s) : launch<__half, __half>(a, form, sms, s);
  return sum_elem == 1 ? launch<__nv_bfloat16, float>(a, form, sms, s) : launch<__nv_bfloat16, __nv_bfloat16>(a, form, sms, s);
}

}  // namespace k
}  // namespace sb
