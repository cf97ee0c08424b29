// What the kernels of paged attention share: operand types, launch arguments, the join of split items.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "decoder.h"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace sb {
namespace k {
namespace {

template <typename T> struct Mma;
template <> struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static constexpr uint32_t kExp = 0x7c00u;   // exponent bits of infinities and NaN
  static __device__ __forceinline__ float widen(uint16_t b) { return __half2float(__ushort_as_half(b)); }
};
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static constexpr uint32_t kExp = 0x7f80u;
  static __device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float(uint32_t(b) << 16); }
};

// The weights of a step of positions are 2^(s - m + kLift), s and m in units of log2, rounded to the operands' type.
// m is a reference near the running maximum, the same for o and l, which are fp32; any value serves that keeps the
// step's own weights within the type. A step's maximum more than kGrowth above m becomes m, so that o is rescaled
// a few times per row only and weights stay below 2^(kLift + kGrowth).
// fp16 has full precision from 2^-14 to 2^15 only, far less than what softmax weights span: after a leading position
// 17 nats above the others all of theirs would be below 2^-24 of it, and thousands of them gone from o but not from
// l. So m is lifted to the top of that range, and brought down to kBack above a step's maximum that is more than
// kFall below it: a step's largest weight is 2^-2 or more, and a weight is off by 2^-11 of itself or 2^-23 of the
// largest of its step. At most kDeepest at a time and while l < kMostSum, so that o (up to 65504 l) stays in
// fp32. A weight that is lost then is below 2^-75 of l, and 2^30 of them with values of 65504 round to zero.
template <typename T> struct Reference {   // bf16: the range of fp32
  static constexpr float kLift = 0.f, kGrowth = 8.f;
  static constexpr bool kFalls = false;
};
template <> struct Reference<__half> {
  static constexpr float kLift = 11.f, kGrowth = 4.f;
  static constexpr bool kFalls = true;
};
constexpr float kFall = 13.f, kBack = 10.f, kDeepest = 40.f, kMostSum = 1125899906842624.f;   // 2^50

// Whether a step whose maximum is `above` (its distance from m) needs another reference. Not where m or the
// maximum is infinite, but for a row's first logits.
template <typename T> __device__ __forceinline__ bool rises(float above) { return above > Reference<T>::kGrowth; }
template <typename T> __device__ __forceinline__ bool falls(float above) {
  return Reference<T>::kFalls && above < -kFall && above > -INFINITY;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A partial result that a cut left: slot 2c is the first piece of CTA c, slot 2c + 1 its last.
struct PartialNote {
  int b, h, i;
  int more;   // > 0: the item begins here and `more` pieces follow in slots 2(c + 1), 2(c + 2), ..; else 0
};

// How long a wait of the chunk kernel may last, and one attempt of it.
struct WaitLimit {
  uint64_t ns;
  uint32_t sleep_ns;
};

struct PagedArgs {
  PagedView c;
  HeadsView q, out;
  int group, window, ctas, least;
  float scale_log2;
  PartialNote* notes;   // [2 * ctas]
  float2* ml;           // [2 * ctas][rows]: m (in units of log2), l
  float* o;             // [2 * ctas][rows][DP]; chunks: [2 * ctas][DP / 4][rows][4]
  WaitLimit wait;       // chunks
};

template <typename F>
cudaError_t launch_dependent(F kernel, dim3 grid, int threads, const PagedArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename F>
cudaError_t allow_smem(F kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (done.load() & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

inline size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// Sizes of a call's workspace parts and its grid.
struct PagedSpace {
  int ctas, dp;
  size_t notes, ml, o;
};
bool paged_chunk_wanted(const PagedView& c);
PagedSpace paged_chunk_space(const PagedView& c, int sms);
cudaError_t paged_chunk(const PagedView& c, int elem, HeadsView q, HeadsView out, float scale, int window, void* ws, int sms,
                        cudaStream_t s);

}  // namespace k
}  // namespace sb
