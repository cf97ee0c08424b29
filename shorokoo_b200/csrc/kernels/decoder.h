// Launch interface of the decoder-layer kernels (rotary.cu, w4.cu, paged_attention.cu, residual_norm.cu, moe.cu,
// sample.cu): what ../decoder.cpp checks and passes on. Arguments are valid when they get here.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace sb {
namespace k {

struct HeadsView {
  void* p;
  int64_t ts, hs;   // elements between tokens, between heads
};

// The paged cache and the step's rows over it (include/shorokoo_b200.h says what they mean).
struct PagedView {
  void *k, *v;
  int64_t kp, kt, kh, vp, vt, vh;   // elements between pages, tokens of a page, heads
  const int32_t* table;
  const int32_t* ctx;
  const int32_t* starts;
  int64_t table_stride;
  int64_t pages;
  int64_t tokens;
  int page_size, max_pages, batch, kv_heads, head_dim, q_heads;
};

struct RotaryView {
  const uint64_t* phases;
  int pairs, interleaved, inverse;
  float magnitude;
};

// elem: ONNX numbering (1 float32, 10 float16, 16 bfloat16)
cudaError_t rotary(HeadsView x, HeadsView y, int elem, int64_t tokens, int heads, int head_dim, const void* positions,
                   int positions64, RotaryView table, int sms, cudaStream_t s);
// q.p null: keys and values alone; table.phases null: no rotation
cudaError_t paged_append(const PagedView& c, int elem, HeadsView k, HeadsView v, HeadsView q, HeadsView q_out,
                         RotaryView table, int sms, cudaStream_t s);

size_t paged_attention_workspace(const PagedView& c, int sms);
cudaError_t paged_attention(const PagedView& c, int elem, HeadsView q, HeadsView out, float scale, int window, void* ws,
                            int sms, cudaStream_t s);

// Waits for the stream; bits of the attention kernels' waits that ran out since the last call.
cudaError_t paged_wait_errors(unsigned* bits, cudaStream_t s);

struct W4View {
  const void* data;
  int64_t n, k;
  int group, zeros, elem;
};
size_t w4_layout_bytes(const W4View& w);
cudaError_t w4_layout(const W4View& w, const uint8_t* packed, int64_t row_bytes, const void* scales, const uint8_t* zeros,
                      void* data, cudaStream_t s);
cudaError_t linear_w4(const W4View& w, const void* x, int64_t xs, const void* bias, void* y, int64_t ys, int64_t rows,
                      int sms, cudaStream_t s);

// Rows of width elements; strides between them in elements. Null: not there.
struct ResidualNormArgs {
  const void *x, *residual, *gate;
  void *sum, *y;
  int64_t xs, rs, gs, ss, ys;
  const void *weight, *bias, *post_weight, *post_bias;
  int64_t rows;
  int width, weight_elem, layer;   // layer: the mean is taken off
  float scale, eps, offset;        // offset: added to the weights
  float per_width;                 // 1 / width, set by residual_norm
};
cudaError_t residual_norm(const ResidualNormArgs& a, int elem, int sum_elem, int sms, cudaStream_t s);

struct MoEView {
  const void *router, *gate_up, *down;   // [experts][width], [experts][2 inner][width], [experts][width][inner]
  const float* selection_bias;           // [experts] or null
  int64_t router_row, up_expert, up_row, down_expert, down_row;
  int elem, router_elem, experts, width, inner, top_k;
  int softmax, normalize, gelu;
  float scale;
};
size_t moe_workspace(const MoEView& w, int64_t tokens);
cudaError_t moe(const MoEView& w, const void* x, int64_t xs, void* y, int64_t ys, int64_t tokens, void* ws, int sms, cudaStream_t s);

constexpr int kMostVocab = 1 << 21;   // logits of a row that sample takes

// Settings of all rows, or (not null) of each.
struct SamplingView {
  const float *temperature_of, *top_p_of, *min_p_of;
  const int32_t* top_k_of;
  float temperature, top_p, min_p;
  int top_k;
};
cudaError_t sample(const void* logits, int64_t stride, int elem, int64_t rows, int vocab, const float* uniform, const SamplingView& by,
                   int64_t* tokens, int sms, cudaStream_t s);

}  // namespace k
}  // namespace sb
