// Rotary positions, and the write of a step's keys and values into a paged cache.
//
// A pair (a, b) of a head turns by t = position * frequency:
//   a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t)        (inverse: -t)
// computed in fp32 and rounded once to the element type. Pairs are (2i, 2i + 1) or (i, i + pairs).
//
// The angle: 32-bit products lose it at far positions (position 10^6 in fp32 is off by 0.06 rad), so a
// frequency is held as the 64-bit binary fraction of a turn per position and the product with the
// position is taken modulo 2^64, that is exactly modulo one turn: the fraction's own rounding costs 2^-65 of a
// turn per position, nothing else grows with it. Its top 32 bits, as a signed number in [-1, 1) half turns, are
// rounded to fp32 for sincospif: about 2^-26 of a turn, 2^-25 pi radians, no more than what the results' own fp32
// products lose (fp32 error against 64 bits 3.8e-8 of the values; 3.0e-8 with angles in 64 bits).
//
// Every value is read and written once: the kernels are bound by memory bandwidth (and, for a decode
// step of some tens of tokens, by launch latency). A CTA takes one or a few tokens: the angles of its
// tokens are computed once into shared memory and used by all their heads, 16-byte pieces per thread.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "decoder.h"
#include "paged.cuh"

namespace sb {
namespace k {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kMostTokensPerCta = 8;

struct RotaryArgs {
  HeadsView q, qo;        // rotated: q_heads
  HeadsView k, v;         // append: kv_heads each, into the cache
  int q_heads, kv_heads;
  int head_dim, pairs;    // pairs 0: nothing turns
  int rot_units, copy_units;
  float magnitude, sign;
  const uint64_t* phases;
  const void* positions;
  int positions64;
  int64_t tokens;
  int per_cta;            // tokens of a CTA
  PagedView c;
};

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float load(float x) { return x; }
  static __device__ __forceinline__ float store(float x) { return x; }
};
template <> struct Elem<__half> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float load(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half store(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float load(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 store(float x) { return __float2bfloat16_rn(x); }
};

template <typename T, int V> struct alignas(V * sizeof(T)) Piece { T e[V]; };

// V: elements per memory access (a 16-byte piece, or 1 where alignment, strides or sizes allow no more)
template <typename T, int V, bool kInter, bool kAppend>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 turns[];   // [per_cta][pairs] magnitude * (cos, sin)
  __shared__ int64_t position[kMostTokensPerCta];
  __shared__ int64_t k_slot[kMostTokensPerCta], v_slot[kMostTokensPerCta];   // element offsets in the cache
  __shared__ int present[kMostTokensPerCta];   // 0: a row of no sequence, 1: without a slot, 3: with one
  const int tid = threadIdx.x;
  const int64_t t0 = int64_t(blockIdx.x) * a.per_cta;
  const int count = int(min(int64_t(a.per_cta), a.tokens - t0));
  const int units = a.rot_units + a.copy_units;
  const int heads = a.q_heads + (kAppend ? 2 * a.kv_heads : 0);
  const int per_token = heads * units;
  const int items = count * per_token, stride = gridDim.y * kRotaryThreads;
  using P = Piece<T, V>;

  // An item: one piece of the copied or interleaved part of a head, or the two of a pair's halves.
  struct Item {
    int w, h, u;      // token of the CTA, head (q, then k, then v), unit of the head
    int ia, ib;       // elements of its pieces in the head; ib < 0: one piece
  };
  auto item = [&](int i) {
    Item it;
    it.w = count == 1 ? 0 : i / per_token;
    const int r = i - it.w * per_token;
    it.h = r / units;
    it.u = r - it.h * units;
    if (it.u >= a.rot_units) it.ia = 2 * a.pairs + (it.u - a.rot_units) * V, it.ib = -1;
    else if (kInter && V > 1) it.ia = it.u * V, it.ib = -1;
    else it.ia = kInter ? 2 * it.u : it.u * V, it.ib = kInter ? 2 * it.u + 1 : a.pairs + it.u * V;
    return it;
  };
  auto fetch = [&](const Item& it, P& xa, P& xb) {
    const int64_t token = t0 + it.w;
    const T* src;
    if (!kAppend || it.h < a.q_heads) src = static_cast<const T*>(a.q.p) + token * a.q.ts + it.h * a.q.hs;
    else if (it.h < a.q_heads + a.kv_heads) src = static_cast<const T*>(a.k.p) + token * a.k.ts + (it.h - a.q_heads) * a.k.hs;
    else src = static_cast<const T*>(a.v.p) + token * a.v.ts + (it.h - a.q_heads - a.kv_heads) * a.v.hs;
    xa = *reinterpret_cast<const P*>(src + it.ia);
    if (it.ib >= 0) xb = *reinterpret_cast<const P*>(src + it.ib);
  };
  auto finish = [&](const Item& it, P& xa, P& xb) {
    if (kAppend && !present[it.w]) return;
    T* dst;
    bool turn = it.u < a.rot_units;
    if (!kAppend || it.h < a.q_heads) {
      dst = static_cast<T*>(a.qo.p) + (t0 + it.w) * a.qo.ts + it.h * a.qo.hs;
    } else {
      if (!(present[it.w] & 2)) return;
      int hk = it.h - a.q_heads;
      if (hk < a.kv_heads) {
        dst = static_cast<T*>(a.c.k) + k_slot[it.w] + hk * a.c.kh;
      } else {
        turn = false;
        hk -= a.kv_heads;
        dst = static_cast<T*>(a.c.v) + v_slot[it.w] + hk * a.c.vh;
      }
    }
    if (turn) {
      if (kInter && V > 1) {
        const float2* cs = turns + it.w * a.pairs + it.ia / 2;
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) {
          const float va = Elem<T>::load(xa.e[e]), vb = Elem<T>::load(xa.e[e + 1]);
          xa.e[e] = Elem<T>::store(va * cs[e / 2].x - vb * cs[e / 2].y);
          xa.e[e + 1] = Elem<T>::store(va * cs[e / 2].y + vb * cs[e / 2].x);
        }
      } else {
        const float2* cs = turns + it.w * a.pairs + it.u * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float va = Elem<T>::load(xa.e[e]), vb = Elem<T>::load(xb.e[e]);
          xa.e[e] = Elem<T>::store(va * cs[e].x - vb * cs[e].y);
          xb.e[e] = Elem<T>::store(va * cs[e].y + vb * cs[e].x);
        }
      }
    }
    *reinterpret_cast<P*>(dst + it.ia) = xa;
    if (it.ib >= 0) *reinterpret_cast<P*>(dst + it.ib) = xb;
  };

  // An append's first item is under way while the slots are looked up (5600 tokens: 41 -> 35 us; two items: 39
  // us, for their registers). Without slots to wait for, the plain loop at the end is as fast or faster (4099
  // tokens of 32 heads of 128: 18.2 us against 18.4 to 19.9, 3.7 TB/s).
  const int first = blockIdx.y * kRotaryThreads + tid;
  Item early;
  P ea, eb;
  if (kAppend && first < items) {
    early = item(first);
    fetch(early, ea, eb);
  }
  if (kAppend) {
    const int w = tid >> 5;
    if (w < count) {
      const int64_t token = t0 + w;
      const int b = find_sequence(a.c, token);
      const SeqRows s = seq_rows(a.c, b);
      const bool in = token >= s.first && token < s.end;
      const int64_t pos = s.ctx - (s.end - token);
      if ((tid & 31) == 0) {
        present[w] = in;
        position[w] = pos;
        int64_t ks = 0, vs = 0;
        if (in && pos >= 0 && pos < int64_t(a.c.max_pages) * a.c.page_size) {
          const int page_no = int(pos / a.c.page_size), row = int(pos - int64_t(page_no) * a.c.page_size);
          const int page = a.c.table[int64_t(b) * a.c.table_stride + page_no];
          if (page >= 0 && page < a.c.pages) {
            ks = page * a.c.kp + row * a.c.kt;
            vs = page * a.c.vp + row * a.c.vt;
            present[w] = 3;
          }
        }
        k_slot[w] = ks;
        v_slot[w] = vs;
      }
    }
  } else {
    if (tid < count) {
      position[tid] = a.positions64 ? static_cast<const int64_t*>(a.positions)[t0 + tid]
                                    : int64_t(static_cast<const int32_t*>(a.positions)[t0 + tid]);
    }
  }
  __syncthreads();
  for (int i = tid; i < count * a.pairs; i += kRotaryThreads) {
    const int w = count == 1 ? 0 : i / a.pairs, p = i - w * a.pairs;
    const uint64_t phase = uint64_t(position[w]) * a.phases[p];
    const float half_turns = float(int32_t(phase >> 32)) * 4.656612873077393e-10f;   // 2^-31
    float sn, cs;
    sincospif(half_turns, &sn, &cs);
    turns[i] = make_float2(a.magnitude * cs, a.magnitude * a.sign * sn);
  }
  __syncthreads();
  if constexpr (kAppend) {
    if (first < items) finish(early, ea, eb);
    for (int i = first + stride; i < items; i += stride) {
      const Item it = item(i);
      P xa, xb;
      fetch(it, xa, xb);
      finish(it, xa, xb);
    }
  } else for (int i = first; i < items; i += stride) {
    const int w = count == 1 ? 0 : i / per_token;
    const int r = i - w * per_token, h = r / units, u = r - h * units;
    const T* src = static_cast<const T*>(a.q.p) + (t0 + w) * a.q.ts + h * a.q.hs;
    T* dst = static_cast<T*>(a.qo.p) + (t0 + w) * a.qo.ts + h * a.qo.hs;
    if (u >= a.rot_units) {   // behind the rotated part
      const int at = 2 * a.pairs + (u - a.rot_units) * V;
      *reinterpret_cast<P*>(dst + at) = *reinterpret_cast<const P*>(src + at);
    } else if (kInter && V > 1) {
      const int at = u * V;
      P x = *reinterpret_cast<const P*>(src + at);
      const float2* cs = turns + w * a.pairs + at / 2;
#pragma unroll
      for (int e = 0; e + 1 < V; e += 2) {
        const float va = Elem<T>::load(x.e[e]), vb = Elem<T>::load(x.e[e + 1]);
        x.e[e] = Elem<T>::store(va * cs[e / 2].x - vb * cs[e / 2].y);
        x.e[e + 1] = Elem<T>::store(va * cs[e / 2].y + vb * cs[e / 2].x);
      }
      *reinterpret_cast<P*>(dst + at) = x;
    } else {
      const int ia = kInter ? 2 * u : u * V, ib = kInter ? 2 * u + 1 : a.pairs + u * V;
      P xa = *reinterpret_cast<const P*>(src + ia), xb = *reinterpret_cast<const P*>(src + ib);
      const float2* cs = turns + w * a.pairs + u * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float va = Elem<T>::load(xa.e[e]), vb = Elem<T>::load(xb.e[e]);
        xa.e[e] = Elem<T>::store(va * cs[e].x - vb * cs[e].y);
        xb.e[e] = Elem<T>::store(va * cs[e].y + vb * cs[e].x);
      }
      *reinterpret_cast<P*>(dst + ia) = xa;
      *reinterpret_cast<P*>(dst + ib) = xb;
    }
  }
}

bool pieces(const HeadsView& h, int vec, size_t bytes) {
  return reinterpret_cast<uintptr_t>(h.p) % bytes == 0 && h.ts % vec == 0 && h.hs % vec == 0;
}

template <typename T, bool kAppend>
cudaError_t launch(RotaryArgs a, bool inter, bool vec, int sms, cudaStream_t s) {
  constexpr int kV = Elem<T>::kVec;
  const int r = 2 * a.pairs, d = a.head_dim;
  vec = vec && d % kV == 0 && (inter ? r : a.pairs) % kV == 0;
  const int v = vec ? kV : 1;
  a.rot_units = vec && inter ? r / kV : a.pairs / v;
  a.copy_units = (d - r) / v;
  const int64_t per_token = int64_t(a.q_heads + (kAppend ? 2 * a.kv_heads : 0)) * (a.rot_units + a.copy_units);
  if (per_token > (int64_t(1) << 27)) return cudaErrorInvalidValue;
  // Tokens of few pieces share a CTA (two pieces per thread) while the card stays full; tokens of many
  // are split over CTAs while it is not. Replayed from a graph: 5000 tokens of 2 heads of 64 in bf16 9.5 us one to a
  // CTA, 3.6 eight to a CTA (1200 tokens: 3.4 and 2.5); 32 tokens of 64 heads of 128 in fp32 5.1 us whole, 3.1 split.
  int per_cta = 1;
  while (per_cta < kMostTokensPerCta && per_cta * 2 * per_token <= 2 * kRotaryThreads &&
         a.tokens >= int64_t(per_cta) * 2 * 4 * sms && int64_t(per_cta) * 2 * a.pairs <= 4096)
    per_cta *= 2;
  a.per_cta = per_cta;
  const int64_t blocks = (a.tokens + per_cta - 1) / per_cta;
  int split = 1;
  while (blocks * split < 2 * sms && per_token * per_cta > int64_t(split) * kRotaryThreads) split *= 2;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min(split, 1024)));
  const size_t smem = size_t(per_cta) * a.pairs * sizeof(float2);
  if (vec && inter) rotary_kernel<T, kV, true, kAppend><<<grid, kRotaryThreads, smem, s>>>(a);
  else if (vec) rotary_kernel<T, kV, false, kAppend><<<grid, kRotaryThreads, smem, s>>>(a);
  else if (inter) rotary_kernel<T, 1, true, kAppend><<<grid, kRotaryThreads, smem, s>>>(a);
  else rotary_kernel<T, 1, false, kAppend><<<grid, kRotaryThreads, smem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t rotary(HeadsView x, HeadsView y, int elem, int64_t tokens, int heads, int head_dim, const void* positions,
                   int positions64, RotaryView table, int sms, cudaStream_t s) {
  RotaryArgs a = {};
  a.q = x, a.qo = y, a.q_heads = heads, a.head_dim = head_dim, a.pairs = table.pairs;
  a.magnitude = table.magnitude, a.sign = table.inverse ? -1.f : 1.f, a.phases = table.phases;
  a.positions = positions, a.positions64 = positions64, a.tokens = tokens;
  const int vec = elem == 1 ? 4 : 8;
  const bool wide = pieces(x, vec, 16) && pieces(y, vec, 16);
  if (elem == 1) return launch<float, false>(a, table.interleaved, wide, sms, s);
  if (elem == 10) return launch<__half, false>(a, table.interleaved, wide, sms, s);
  return launch<__nv_bfloat16, false>(a, table.interleaved, wide, sms, s);
}

cudaError_t paged_append(const PagedView& c, int elem, HeadsView k, HeadsView v, HeadsView q, HeadsView q_out,
                         RotaryView table, int sms, cudaStream_t s) {
  RotaryArgs a = {};
  a.q = q, a.qo = q_out, a.k = k, a.v = v, a.q_heads = q.p ? c.q_heads : 0, a.kv_heads = c.kv_heads;
  a.head_dim = c.head_dim, a.pairs = table.pairs, a.magnitude = table.magnitude, a.sign = 1.f, a.phases = table.phases;
  a.tokens = c.tokens, a.c = c;
  const bool wide = pieces(k, 8, 16) && pieces(v, 8, 16) && pieces({c.k, c.kt, c.kh}, 8, 16) && pieces({c.v, c.vt, c.vh}, 8, 16) &&
                    c.kp % 8 == 0 && c.vp % 8 == 0 && (!q.p || (pieces(q, 8, 16) && pieces(q_out, 8, 16)));
  if (elem == 10) return launch<__half, true>(a, table.interleaved, wide, sms, s);
  return launch<__nv_bfloat16, true>(a, table.interleaved, wide, sms, s);
}

}  // namespace k
}  // namespace sb
