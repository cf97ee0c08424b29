// Linear layer with 4-bit weights for few rows: y[m, n] = sum_k x[m, k] (c[n, k] - z[n, k/g]) s[n, k/g] + b[n].
//
// One row of inputs needs 2 K operations per K / 2 bytes of weights: the weights' bytes bound it (HBM,
// or L2 where they stay there). The products still go to the tensor core (mma m16n8k16, fp32
// accumulators): 16 outputs x 8 rows per instruction costs no more than one row would, and takes the
// multiply-adds off the issue slots, which turning codes into operands needs (about one instruction
// per weight). c - z is a small integer and exact in either 16-bit type; the group's scale is applied
// in fp32 to the products' sum over a group, so nothing is rounded but x (given in 16 bits) and y.
//
// Layout (w4_layout): tiles of 16 outputs x 64 inputs, 512 bytes each, K running fastest: one 16-byte
// load per lane is the whole warp's operand for four k16 steps, with all 16 inputs of a step in one
// group of 32. Lane 4g + t holds outputs g and g + 8, inputs 8t .. 8t + 7 of both 32-input halves, one
// word each; nibble i and nibble 4 + i of a word are inputs 2i and 2i + 1, so that shifting by 4i and
// masking gives a register of the operand with its neighbouring pair, and x needs no reordering.
// Inputs past K and outputs past N are zero codes; x reads as zero there. Behind the tiles, scales
// as pairs (output g, g + 8), each pair's groups in a row; then zero points likewise.
//
// A CTA computes 16 or 32 outputs: its warps take the 64-input blocks in turn and their sums meet in shared
// memory, added in a fixed order. One row has a kernel of its own.
//
// Measured (8192 inputs, 22016 outputs, groups of 32 with zero points, fp16, 104 MB): one row 31 us, 3.4 TB/s,
// 0.52 of the measured HBM rate (its loads alone take 27 us, its arithmetic alone about 14 us of issue slots);
// with the kernel for several rows 51 us. 13 rows by 4096 inputs and 11000 outputs, groups of 64, zero points: 21 us
// (19.6 replayed from a graph); 125 registers leave two CTAs per SM, so that its 344 CTAs take two waves.
// The figures at the choices below are replayed from a graph, 4096 inputs, weights from HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "decoder.h"

namespace sb {
namespace k {
namespace {

struct W4Args {
  const uint4* w;
  const uint32_t* scales;   // [tile][8][pitch] pairs
  const uint16_t* zeros;    // [tile][8][pitch] pairs of bytes
  const void* x;
  const void* bias;
  void* y;
  int64_t xs, ys, rows, n, k;
  int blocks, groups, group;
  int pitch;   // groups, in whole eights
  int shift;   // log2 of the group size, or -1
};

struct W4Sizes {
  int64_t tiles, blocks, groups, pitch;
  size_t w, s, z;
};
W4Sizes sizes(const W4View& w) {
  W4Sizes z;
  z.tiles = (w.n + 15) / 16;
  z.blocks = (w.k + 63) / 64;
  z.groups = (w.k + w.group - 1) / w.group;
  z.pitch = (z.groups + 7) / 8 * 8;
  z.w = size_t(z.tiles) * z.blocks * 512;
  z.s = size_t(z.tiles) * z.pitch * 32;
  z.z = w.zeros ? size_t(z.tiles) * z.pitch * 16 : 0;
  return z;
}

template <typename T> struct Half;
template <> struct Half<__half> {
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  static __device__ __forceinline__ float2 both(uint32_t a) { return __half22float2(*reinterpret_cast<__half2*>(&a)); }
  static __device__ __forceinline__ float one(__half a) { return __half2float(a); }
  static __device__ __forceinline__ __half round(float a) { return __float2half_rn(a); }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  static __device__ __forceinline__ float2 both(uint32_t a) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&a));
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 a) { return __bfloat162float(a); }
  static __device__ __forceinline__ __nv_bfloat16 round(float a) { return __float2bfloat16_rn(a); }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// (Volatile like the codes', or the compiler moves these loads down to their use, behind their latency.)
__device__ __forceinline__ uint32_t load_scales(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t load_zeros(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}

// 8 inputs from element k of a row (zero past K); kWide: K, the row stride and the address allow 16 bytes
template <bool kWide>
__device__ __forceinline__ uint4 load_x(const uint16_t* row, int k, int kmax) {
  if (kWide) return k < kmax ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = k + 2 * i < kmax ? row[k + 2 * i] : 0, hi = k + 2 * i + 1 < kmax ? row[k + 2 * i + 1] : 0;
    w[i] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kW4Warps = 8;

// What a warp reads of a 64-input block besides x, and has in flight for the blocks to come.
struct Block {
  uint4 w;
  uint2 s;       // scale pairs (output g, g + 8) of the two halves
  uint2 z;       // their zero points, a byte each
};

template <typename T> struct Codes;
// Operand registers of 8 codes less their zero point. magic + code is exact in the type; fp16's 10 mantissa bits
// also hold a code four bits up (1024 + 16 code), which saves the shift.
template <> struct Codes<__nv_bfloat16> {
  // magic + zero point of byte `which` of z, twice
  static __device__ __forceinline__ uint32_t zero(uint32_t z, int which) { return __byte_perm(z, 0x43u, 0x4040u | uint32_t(which * 0x0101)); }
  static __device__ __forceinline__ void spread(uint32_t w, uint32_t z, uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = Half<__nv_bfloat16>::sub(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u, z);
  }
};
template <> struct Codes<__half> {
  static __device__ __forceinline__ uint32_t zero(uint32_t z, int which) { return __byte_perm(z, 0x64u, 0x4040u | uint32_t(which * 0x0101)); }
  static __device__ __forceinline__ void spread(uint32_t w, uint32_t z, uint32_t (&r)[4]) {
    const __half2 z1 = *reinterpret_cast<__half2*>(&z);
    // (1024 + 16 c) / 16 - (64 + z) = c - z, where 64 + z = (1024 + z) - 960
    const __half2 z16 = __hsub2(__float2half2_rn(960.f), z1), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = w >> (8 * i);
      r[2 * i] = Half<__half>::sub((v & 0x000f000fu) | 0x64006400u, z);
      uint32_t up = (v & 0x00f000f0u) | 0x64006400u;
      const __half2 d = __hfma2(*reinterpret_cast<__half2*>(&up), sixteenth, z16);
      r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
};

// MT: row tiles of 8; TN: 16-output tiles of a CTA; kPerBlock: one group covers a 64-input block (else one
// per 32).
template <typename T, int MT, int TN, bool kZeros, bool kPerBlock, bool kWide>
__global__ void __launch_bounds__(kW4Warps * 32) linear_w4_kernel(const W4Args a) {
  constexpr int kDepth = 4 / TN;           // blocks in flight per warp and tile
  constexpr int kAhead = MT <= 2 ? 1 : 0;  // blocks that x is read ahead
  __shared__ float sums[kW4Warps][TN * 16][MT * 8 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t tile0 = int64_t(blockIdx.x) * TN, m0 = int64_t(blockIdx.y) * (MT * 8);
  const uint4* w[TN];
  const uint32_t* scales[TN];
  const uint16_t* zeros[TN];
#pragma unroll
  for (int n = 0; n < TN; ++n) {
    const int64_t tile = min(tile0 + n, (a.n + 15) / 16 - 1);   // a tile past the last one repeats it, unstored
    w[n] = a.w + tile * a.blocks * 32 + lane;
    scales[n] = a.scales + (tile * 8 + g) * a.pitch;
    zeros[n] = a.zeros + (tile * 8 + g) * a.pitch;
  }
  const uint16_t* x[MT];
  bool live[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + i * 8 + g;
    live[i] = m < a.rows;
    x[i] = static_cast<const uint16_t*>(a.x) + (live[i] ? m : m0) * a.xs + t * 8;
  }
  const int kmax = int(a.k) - t * 8;   // of this lane's pieces of x
  auto load = [&](Block (&b)[TN], int kb) {
    const int g0 = a.shift >= 0 ? (kb * 64) >> a.shift : kb * 64 / a.group;
    int g1 = 0;
    if (!kPerBlock)   // the last block's second half may lie past K
      g1 = min(a.shift >= 0 ? (kb * 64 + 32) >> a.shift : (kb * 64 + 32) / a.group, a.groups - 1);
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      b[n].w = load_once(w[n] + int64_t(kb) * 32);
      b[n].s.x = load_scales(scales[n] + g0);
      if (kZeros) b[n].z.x = load_zeros(zeros[n] + g0);
      if (!kPerBlock) {
        b[n].s.y = load_scales(scales[n] + g1);
        if (kZeros) b[n].z.y = load_zeros(zeros[n] + g1);
      }
    }
  };
  auto load_rows = [&](uint4 (&v)[MT][2], int kb) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        v[i][half] = live[i] ? load_x<kWide>(x[i], kb * 64 + half * 32, kmax) : make_uint4(0, 0, 0, 0);
  };
  float acc[TN][MT][4];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;

  Block next[kDepth][TN];
  uint4 xn[MT][2];
#pragma unroll
  for (int j = 0; j < kDepth; ++j)
    if (warp + j * kW4Warps < a.blocks) load(next[j], warp + j * kW4Warps);
  if (kAhead && warp < a.blocks) load_rows(xn, warp);
  for (int kb0 = warp; kb0 < a.blocks; kb0 += kW4Warps * kDepth) {
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      const int kb = kb0 + j * kW4Warps;
      if (kb < a.blocks) {
        Block b[TN];
        uint4 xv[MT][2];
#pragma unroll
        for (int n = 0; n < TN; ++n) b[n] = next[j][n];
        if (kAhead) {
#pragma unroll
          for (int i = 0; i < MT; ++i) xv[i][0] = xn[i][0], xv[i][1] = xn[i][1];
          if (kb + kW4Warps < a.blocks) load_rows(xn, kb + kW4Warps);
        } else {
          load_rows(xv, kb);
        }
        if (kb + kW4Warps * kDepth < a.blocks) load(next[j], kb + kW4Warps * kDepth);
#pragma unroll
        for (int n = 0; n < TN; ++n) {
          const uint32_t word[4] = {b[n].w.x, b[n].w.y, b[n].w.z, b[n].w.w};
          float part[MT][4];
          uint32_t z0 = Codes<T>::zero(8u, 0), z1 = z0;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half == 0 || !kPerBlock) {
#pragma unroll
              for (int i = 0; i < MT; ++i) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.f;
              if (kZeros) {
                z0 = Codes<T>::zero(half ? b[n].z.y : b[n].z.x, 0);
                z1 = Codes<T>::zero(half ? b[n].z.y : b[n].z.x, 1);
              }
            }
            uint32_t lo[4], hi[4];   // outputs g and g + 8
            Codes<T>::spread(word[2 * half], z0, lo);
            Codes<T>::spread(word[2 * half + 1], z1, hi);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const uint4 v = xv[i][half];
              Half<T>::mma(part[i], lo[0], hi[0], lo[1], hi[1], v.x, v.y);
              Half<T>::mma(part[i], lo[2], hi[2], lo[3], hi[3], v.z, v.w);
            }
            if (half == 1 || !kPerBlock) {
              const float2 s = Half<T>::both(!kPerBlock && half == 1 ? b[n].s.y : b[n].s.x);
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                acc[n][i][0] += s.x * part[i][0];
                acc[n][i][1] += s.x * part[i][1];
                acc[n][i][2] += s.y * part[i][2];
                acc[n][i][3] += s.y * part[i][3];
              }
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      sums[warp][n * 16 + g][i * 8 + 2 * t] = acc[n][i][0];
      sums[warp][n * 16 + g][i * 8 + 2 * t + 1] = acc[n][i][1];
      sums[warp][n * 16 + g + 8][i * 8 + 2 * t] = acc[n][i][2];
      sums[warp][n * 16 + g + 8][i * 8 + 2 * t + 1] = acc[n][i][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < TN * 16 * MT * 8; i += kW4Warps * 32) {
    const int r = i % (TN * 16), col = i / (TN * 16);
    const int64_t n = tile0 * 16 + r, m = m0 + col;
    if (n >= a.n || m >= a.rows) continue;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kW4Warps; ++j) s += sums[j][r][col];
    if (a.bias) s += Half<T>::one(static_cast<const T*>(a.bias)[n]);
    static_cast<T*>(a.y)[m * a.ys + n] = Half<T>::round(s);
  }
}

// One row of x, groups of 32, 64, 128 or whole 256s. The 8 columns of the products, which 8 rows would use,
// keep 8 groups of 32 inputs apart: a step's x stands in the column of its group, the others are zero. So 256
// inputs go through the tensor core before their scales are applied, once, and lane 4g + t, which holds columns
// 2t and 2t + 1, needs just the scales of those; and x is one 16-byte load per lane for all of them. Against
// the kernel for several rows, 62 instead of 110 instructions per 64-input block.
template <typename T, bool kZeros, bool kWide>
__global__ void __launch_bounds__(256) linear_w4_row_kernel(const W4Args a) {
  __shared__ float sums[8][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warps = blockDim.x >> 5;
  const int64_t tile = blockIdx.x;
  const uint4* w = a.w + tile * a.blocks * 32 + lane;
  const uint32_t* scales = a.scales + (tile * 8 + g) * a.pitch;
  const uint16_t* zeros = a.zeros + (tile * 8 + g) * a.pitch;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + g * 32 + t * 8;
  const int kmax = int(a.k) - (g * 32 + t * 8), supers = (a.blocks + 3) / 4;
  struct Super {
    uint4 w[4], x, z;
    uint2 s;
  };
  auto load = [&](Super& v, int sb) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v.w[j] = sb * 4 + j < a.blocks ? load_once(w + (sb * 4 + j) * 32) : make_uint4(0, 0, 0, 0);
    v.x = load_x<kWide>(x, sb * 256, kmax);
    if (a.shift == 5) {
      const int gi = sb * 8;
      asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.s.x), "=r"(v.s.y) : "l"(scales + gi + 2 * t));
      if (kZeros)
        asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v.z.x), "=r"(v.z.y), "=r"(v.z.z), "=r"(v.z.w) : "l"(zeros + gi));
    } else {
      // two columns share a group; groups past the last one have zero codes and x
      v.s.x = v.s.y = load_scales(scales + min((sb * 256 + 64 * t) >> a.shift, a.groups - 1));
      if (kZeros) {
        uint32_t z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = load_zeros(zeros + min((sb * 256 + 64 * j) >> a.shift, a.groups - 1)) * 0x00010001u;
        v.z = make_uint4(z[0], z[1], z[2], z[3]);
      }
    }
  };
  float acc[2] = {0.f, 0.f};
  Super next;
  if (warp < supers) load(next, warp);
  for (int sb = warp; sb < supers; sb += warps) {
    const Super v = next;
    if (sb + warps < supers) load(next, sb + warps);
    const uint32_t zs[4] = {v.z.x, v.z.y, v.z.z, v.z.w};
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t z0 = Codes<T>::zero(8u, 0), z1 = z0;
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      if (kZeros) {
        z0 = Codes<T>::zero(zs[h >> 1], 2 * (h & 1));
        z1 = Codes<T>::zero(zs[h >> 1], 2 * (h & 1) + 1);
      }
      const uint4 c = v.w[h >> 1];
      uint32_t lo[4], hi[4];
      Codes<T>::spread(h & 1 ? c.z : c.x, z0, lo);
      Codes<T>::spread(h & 1 ? c.w : c.y, z1, hi);
      const bool mine = g == h;
      Half<T>::mma(part, lo[0], hi[0], lo[1], hi[1], mine ? v.x.x : 0u, mine ? v.x.y : 0u);
      Half<T>::mma(part, lo[2], hi[2], lo[3], hi[3], mine ? v.x.z : 0u, mine ? v.x.w : 0u);
    }
    const float2 s0 = Half<T>::both(v.s.x), s1 = Half<T>::both(v.s.y);
    acc[0] += s0.x * part[0];
    acc[0] += s1.x * part[1];
    acc[1] += s0.y * part[2];
    acc[1] += s1.y * part[3];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    acc[i] += __shfl_xor_sync(~0u, acc[i], 1);
    acc[i] += __shfl_xor_sync(~0u, acc[i], 2);
    if (t == 0) sums[warp][g + 8 * i] = acc[i];
  }
  __syncthreads();
  const int64_t n = tile * 16 + threadIdx.x;
  if (threadIdx.x < 16 && n < a.n) {
    float s = 0.f;
    for (int j = 0; j < warps; ++j) s += sums[j][threadIdx.x];
    if (a.bias) s += Half<T>::one(static_cast<const T*>(a.bias)[n]);
    static_cast<T*>(a.y)[n] = Half<T>::round(s);
  }
}

__global__ void w4_layout_kernel(const uint8_t* packed, int64_t row_bytes, const uint16_t* scales, const uint8_t* zeros, int64_t n,
                                 int64_t k, int64_t tiles, int64_t blocks, int64_t groups, int64_t pitch, uint32_t* out_w, uint16_t* out_s,
                                 uint8_t* out_z) {
  const int64_t words = tiles * blocks * 128, pairs = tiles * pitch * 16;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < words + pairs; i += int64_t(gridDim.x) * blockDim.x) {
    if (i < words) {
      const int part = int(i & 3), lane = int((i >> 2) & 31);
      const int64_t tb = i >> 7, tile = tb / blocks, kb = tb - tile * blocks;
      const int64_t row = tile * 16 + (lane >> 2) + (part & 1) * 8;
      const int64_t k0 = kb * 64 + (part >> 1) * 32 + (lane & 3) * 8;
      uint32_t word = 0;
      for (int e = 0; e < 8; ++e) {
        const int64_t kk = k0 + e;
        if (row >= n || kk >= k) break;
        const uint32_t byte = packed[row * row_bytes + kk / 2];
        const uint32_t code = (kk & 1) ? byte >> 4 : byte & 15u;
        word |= code << (4 * ((e >> 1) + 4 * (e & 1)));
      }
      out_w[i] = word;
    } else {
      const int64_t j = i - words;
      const int which = int(j & 1);
      const int64_t row_pair = (j >> 1) / pitch, gi = (j >> 1) - row_pair * pitch;
      const int64_t row = (row_pair >> 3) * 16 + (row_pair & 7) + which * 8;
      const bool there = row < n && gi < groups;
      out_s[j] = there ? scales[row * groups + gi] : 0;
      if (zeros) out_z[j] = there ? (zeros[row * groups + gi] & 15) : 0;
    }
  }
}

template <typename T, int MT, int TN, bool kZeros>
cudaError_t launch(const W4Args& a, bool per_block, bool wide, dim3 grid, cudaStream_t s) {
  const int threads = kW4Warps * 32;
  if (per_block && wide) linear_w4_kernel<T, MT, TN, kZeros, true, true><<<grid, threads, 0, s>>>(a);
  else if (per_block) linear_w4_kernel<T, MT, TN, kZeros, true, false><<<grid, threads, 0, s>>>(a);
  else if (wide) linear_w4_kernel<T, MT, TN, kZeros, false, true><<<grid, threads, 0, s>>>(a);
  else linear_w4_kernel<T, MT, TN, kZeros, false, false><<<grid, threads, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T, int MT, int TN>
cudaError_t launch(const W4Args& a, bool zeros, bool per_block, bool wide, cudaStream_t s) {
  const int64_t tiles = (a.n + 15) / 16, per = MT * 8;
  // grid.y covers 65535 row blocks per launch
  for (int64_t m = 0; m < a.rows; m += 65535 * per) {
    W4Args b = a;
    b.rows = std::min(a.rows - m, 65535 * per);
    b.x = static_cast<const uint16_t*>(a.x) + m * a.xs;
    b.y = static_cast<uint16_t*>(a.y) + m * a.ys;
    const dim3 grid(unsigned((tiles + TN - 1) / TN), unsigned((b.rows + per - 1) / per));
    const cudaError_t e =
        zeros ? launch<T, MT, TN, true>(b, per_block, wide, grid, s) : launch<T, MT, TN, false>(b, per_block, wide, grid, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
template <typename T>
cudaError_t launch_row(const W4Args& a, bool zeros, bool wide, int sms, cudaStream_t s) {
  const int64_t tiles = (a.n + 15) / 16;
  const int supers = (a.blocks + 3) / 4;
  // Small CTAs end at different times and leave no SM idle; where there are few of them, more warps per tile. Groups
  // of 128: 22016 outputs 19.0 us with four warps, 22.2 with eight; 4096 outputs 6.4 and 6.0. (Between, four are ahead
  // already: 11000 outputs 11.1 and 12.7.)
  const int threads = 32 * std::max(1, std::min(tiles >= 8 * sms ? 4 : 8, supers));
  const unsigned grid = unsigned(tiles);
  if (zeros && wide) linear_w4_row_kernel<T, true, true><<<grid, threads, 0, s>>>(a);
  else if (zeros) linear_w4_row_kernel<T, true, false><<<grid, threads, 0, s>>>(a);
  else if (wide) linear_w4_row_kernel<T, false, true><<<grid, threads, 0, s>>>(a);
  else linear_w4_row_kernel<T, false, false><<<grid, threads, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch(const W4Args& a, bool zeros, bool per_block, bool wide, int sms, cudaStream_t s) {
  if (a.rows == 1 && a.shift >= 5) return launch_row<T>(a, zeros, wide, sms, s);
  if (a.rows <= 8) {
    // Two tiles of outputs per CTA share the loads of x, where that leaves several CTAs per SM: 8 rows, 22016 outputs,
    // groups of 128, 18.8 us against 23.5 with one; 4 rows with zero points, groups of 64, 24.4 and 24.3 there, 23.5
    // and 20.6 at 19000 outputs, 16.2 and 13.5 at 11000.
    if ((a.n + 31) / 32 >= 4 * sms) return launch<T, 1, 2>(a, zeros, per_block, wide, s);
    return launch<T, 1, 1>(a, zeros, per_block, wide, s);
  }
  if (a.rows <= 16) {
    // ... and here half of what the SMs read of x. 13 rows with zero points, groups of 64: 11000 outputs 19.6 us
    // against 22.8 with one tile, 16384 outputs 22.6 and 30.3, but 4096 outputs 10.2 and 9.7.
    if ((a.n + 31) / 32 >= 2 * sms) return launch<T, 2, 2>(a, zeros, per_block, wide, s);
    return launch<T, 2, 1>(a, zeros, per_block, wide, s);
  }
  // 11000 outputs, groups of 64: 17 rows 24.5 us, 32 rows 28.2; as two passes of 16 rows 38.2 and 40.1
  return launch<T, 4, 1>(a, zeros, per_block, wide, s);
}

}  // namespace

size_t w4_layout_bytes(const W4View& w) {
  const W4Sizes z = sizes(w);
  return z.w + z.s + z.z;
}

cudaError_t w4_layout(const W4View& w, const uint8_t* packed, int64_t row_bytes, const void* scales, const uint8_t* zeros,
                      void* data, cudaStream_t s) {
  const W4Sizes z = sizes(w);
  uint8_t* p = static_cast<uint8_t*>(data);
  const int64_t items = z.tiles * (z.blocks * 128 + z.pitch * 16);
  const unsigned grid = unsigned(std::min<int64_t>((items + 255) / 256, 148 * 32));
  w4_layout_kernel<<<grid, 256, 0, s>>>(packed, row_bytes, static_cast<const uint16_t*>(scales), zeros, w.n, w.k, z.tiles, z.blocks,
                                        z.groups, z.pitch, reinterpret_cast<uint32_t*>(p), reinterpret_cast<uint16_t*>(p + z.w),
                                        p + z.w + z.s);
  return cudaGetLastError();
}

cudaError_t linear_w4(const W4View& w, const void* x, int64_t xs, const void* bias, void* y, int64_t ys, int64_t rows, int sms,
                      cudaStream_t s) {
  const W4Sizes z = sizes(w);
  const uint8_t* p = static_cast<const uint8_t*>(w.data);
  W4Args a;
  a.w = reinterpret_cast<const uint4*>(p);
  a.scales = reinterpret_cast<const uint32_t*>(p + z.w);
  a.zeros = reinterpret_cast<const uint16_t*>(p + z.w + z.s);
  a.x = x, a.bias = bias, a.y = y, a.xs = xs, a.ys = ys, a.rows = rows, a.n = w.n, a.k = w.k;
  a.blocks = int(z.blocks), a.groups = int(z.groups), a.pitch = int(z.pitch), a.group = w.group;
  a.shift = (w.group & (w.group - 1)) == 0 ? __builtin_ctz(unsigned(w.group)) : -1;
  const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && w.k % 8 == 0 && (xs % 8 == 0 || rows == 1);
  const bool per_block = w.group % 64 == 0;
  if (w.elem == 10) return launch<__half>(a, w.zeros, per_block, wide, sms, s);
  return launch<__nv_bfloat16>(a, w.zeros, per_block, wide, sms, s);
}

}  // namespace k
}  // namespace sb
