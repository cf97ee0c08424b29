// extern "C" entry points of the decoder-layer operators (include/shorokoo_b200.h): argument checks,
// the rotary frequency tables, and the hand-over to the kernels. Nothing here allocates or waits.
#include "../../include/shorokoo_b200.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <string>

#include "common.h"
#include "kernels/decoder.h"

namespace sb {
void set_thread_error(const std::string& msg);
}

namespace {

using namespace sb;

template <typename F>
int32_t checked(const char* who, F&& f) {
  try {
    set_thread_error("");
    f();
    return SB_STATUS_OK;
  } catch (const Error& e) {
    set_thread_error(std::string(who) + ": " + e.what());
    return e.code;
  } catch (const std::bad_alloc&) {
    return SB_STATUS_OUT_OF_MEMORY;
  } catch (const std::exception& e) {
    set_thread_error(std::string(who) + ": " + e.what());
    return SB_STATUS_INTERNAL;
  }
}

void need(bool ok, const std::string& msg) { SB_CHECK(ok, SB_INVALID_ARGUMENT, msg); }
void supported(bool ok, const std::string& msg) { SB_CHECK(ok, SB_UNSUPPORTED, msg); }

void launched(cudaError_t e) {
  SB_CHECK(e == cudaSuccess, e == cudaErrorMemoryAllocation ? SB_OUT_OF_MEMORY : SB_CUDA_ERROR,
           std::string(cudaGetErrorString(e)));
}

int multiprocessors() {
  static std::atomic<int> count[64];
  int dev = 0;
  SB_CHECK(cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64, SB_CUDA_ERROR, "no current CUDA device");
  int n = count[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  SB_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0, SB_CUDA_ERROR,
           "cannot read the multiprocessor count");
  count[dev].store(n, std::memory_order_relaxed);
  return n;
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// No buffer of a device spans as many elements, so that a stride beyond is a mistake.
constexpr int64_t kMostStride = int64_t(1) << 40;
bool usable(int64_t stride) { return stride > -kMostStride && stride < kMostStride; }
constexpr int64_t kMostTokens = int64_t(1) << 30;

k::HeadsView view(const sb_heads* h, const char* name, size_t esz) {
  need(h != nullptr && h->data != nullptr, std::string(name) + " is null");
  need(aligned(h->data, esz), std::string(name) + " is not aligned to its element type");
  need(usable(h->token_stride) && usable(h->head_stride),
       std::string(name) + ": stride out of range");
  return {h->data, h->token_stride, h->head_stride};
}

// A result's: writes of the same element by several rows would leave any of them.
void apart(const k::HeadsView& v, const char* name, int64_t tokens, int64_t heads, int64_t head_dim) {
  if ((tokens > 1 && std::llabs(v.ts) < head_dim) || (heads > 1 && std::llabs(v.hs) < head_dim))
    need(false, std::string("rows of ") + name + " overlap");
}

void wide(const k::HeadsView& h, const char* name) {
  supported(aligned(h.p, 16) && h.ts % 8 == 0 && h.hs % 8 == 0,
            std::string(name) + " needs 16-byte alignment and strides of whole 8-element pieces");
}

k::RotaryView view(const sb_rotary_table* t, int head_dim, bool inverse) {
  need(t->phases != nullptr && aligned(t->phases, 8), "table phases are null or misaligned");
  need(t->pairs > 0 && 2 * int64_t(t->pairs) <= head_dim,
       "table has " + std::to_string(t->pairs) + " pairs for a head of " + std::to_string(head_dim));
  supported(t->pairs <= 4096, "more than 4096 rotary pairs");
  need(t->interleaved == 0 || t->interleaved == 1, "table interleaved must be 0 or 1");
  return {t->phases, t->pairs, t->interleaved, inverse ? 1 : 0, t->magnitude};
}

k::PagedView view(const sb_paged_cache* c, int32_t q_heads, int64_t tokens, const int32_t* starts) {
  need(c != nullptr, "cache is null");
  supported(c->elem_type == DT_FLOAT16 || c->elem_type == DT_BFLOAT16,
            std::string("cache element type ") + dtype_name(c->elem_type) + " (float16 or bfloat16)");
  need(c->batch >= 0 && c->max_pages >= 0 && c->pages >= 0 && c->page_size > 0 && c->kv_heads > 0 && c->head_dim > 0,
       "cache sizes must be positive");
  need(c->pages < (int64_t(1) << 31), "more than 2^31 - 1 pages");
  need(int64_t(c->max_pages) * c->page_size <= (int64_t(1) << 30), "more than 2^30 positions per sequence");
  need(c->k != nullptr && c->v != nullptr, "cache k or v is null");
  need((c->page_table != nullptr && c->context_lengths != nullptr) || c->batch == 0, "cache page_table or context_lengths is null");
  need(aligned(c->page_table, 4) && aligned(c->context_lengths, 4), "cache page_table or context_lengths is misaligned");
  need(aligned(c->k, 2) && aligned(c->v, 2), "cache k or v is misaligned");
  for (int64_t s : {c->k_page_stride, c->k_token_stride, c->k_head_stride, c->v_page_stride, c->v_token_stride,
                    c->v_head_stride, c->page_table_stride})
    need(usable(s), "cache stride out of range");
  need(tokens >= 0 && tokens <= kMostTokens, "token count out of range");
  need((starts != nullptr && aligned(starts, 4)) || tokens == 0 || c->batch == 0, "query_starts is null or misaligned");
  k::PagedView p;
  p.k = c->k, p.v = c->v;
  p.kp = c->k_page_stride, p.kt = c->k_token_stride, p.kh = c->k_head_stride;
  p.vp = c->v_page_stride, p.vt = c->v_token_stride, p.vh = c->v_head_stride;
  p.table = c->page_table, p.ctx = c->context_lengths, p.starts = starts;
  p.table_stride = c->page_table_stride, p.pages = c->pages, p.tokens = tokens;
  p.page_size = c->page_size, p.max_pages = c->max_pages, p.batch = c->batch;
  p.kv_heads = c->kv_heads, p.head_dim = c->head_dim, p.q_heads = q_heads;
  return p;
}

// attention's own demands on sizes
void check_attention(const k::PagedView& p) {
  need(p.q_heads > 0 && p.q_heads % p.kv_heads == 0,
       std::to_string(p.q_heads) + " query heads are not a multiple of " + std::to_string(p.kv_heads) + " key heads");
  supported(p.head_dim % 8 == 0 && p.head_dim <= 128,
            "head_dim " + std::to_string(p.head_dim) + " (a multiple of 8 up to 128)");
  // the kernels count a sequence's rows in 32 bits, in steps of up to 32 tiles past the last one
  need(p.tokens * (p.q_heads / p.kv_heads) <= (int64_t(1) << 30), "more than 2^30 tokens x query heads of a key head");
}

k::W4View view(const sb_w4_weights* w) {
  need(w != nullptr, "weights are null");
  supported(w->elem_type == DT_FLOAT16 || w->elem_type == DT_BFLOAT16,
            std::string("element type ") + dtype_name(w->elem_type) + " (float16 or bfloat16)");
  need(w->out_features > 0 && w->in_features > 0 && w->out_features < (int64_t(1) << 31) && w->in_features < (int64_t(1) << 31),
       "features must be positive and below 2^31");
  supported(w->group_size > 0 && w->group_size % 32 == 0, "group_size " + std::to_string(w->group_size) + " (a multiple of 32)");
  return {w->data, w->out_features, w->in_features, w->group_size, w->has_zeros ? 1 : 0, w->elem_type};
}

}  // namespace

extern "C" {

int32_t sb_rotary_frequencies(int32_t rotary_dim, double base, int32_t scaling, double factor, double original_context,
                              double beta_fast, double beta_slow, double* frequencies, double* magnitude) {
  return checked("sb_rotary_frequencies", [&] {
    need(frequencies != nullptr && magnitude != nullptr, "null output");
    need(rotary_dim >= 2 && rotary_dim % 2 == 0, "rotary_dim must be even and positive");
    need(std::isfinite(base) && base > 0, "base must be positive");
    need(scaling >= SB_ROTARY_PLAIN && scaling <= SB_ROTARY_BY_PARTS, "unknown scaling");
    if (scaling != SB_ROTARY_PLAIN) need(std::isfinite(factor) && factor > 0, "factor must be positive");
    if (scaling == SB_ROTARY_NTK) {
      need(rotary_dim > 2, "this scaling needs rotary_dim > 2");
      base *= std::pow(factor, rotary_dim / (rotary_dim - 2.0));
    }
    if (scaling == SB_ROTARY_BY_PARTS) {
      need(factor >= 1, "factor must be at least 1");
      need(std::isfinite(original_context) && original_context > 0, "original_context must be positive");
      need(std::isfinite(beta_fast) && std::isfinite(beta_slow) && beta_fast > beta_slow, "beta_fast must exceed beta_slow");
    }
    *magnitude = scaling == SB_ROTARY_BY_PARTS ? 0.1 * std::log(factor) + 1.0 : 1.0;
    for (int32_t i = 0; i < rotary_dim / 2; ++i) {
      double f = std::pow(base, -2.0 * i / rotary_dim);
      if (scaling == SB_ROTARY_LINEAR) f /= factor;
      if (scaling == SB_ROTARY_BY_PARTS) {
        const double turns = original_context * f / 6.283185307179586477;
        const double keep = std::min(1.0, std::max(0.0, (turns - beta_slow) / (beta_fast - beta_slow)));
        f *= keep + (1.0 - keep) / factor;
      }
      frequencies[i] = f;
    }
  });
}

int32_t sb_rotary_phases(const double* frequencies, int32_t pairs, uint64_t* phases) {
  return checked("sb_rotary_phases", [&] {
    need(frequencies != nullptr && phases != nullptr && pairs > 0, "null array or no pairs");
    for (int32_t i = 0; i < pairs; ++i) need(std::isfinite(frequencies[i]), "frequency is not finite");
    for (int32_t i = 0; i < pairs; ++i) {
      // the long double quotient keeps the 64-bit fraction's own rounding the largest error
      const long double turns = static_cast<long double>(frequencies[i]) / 6.283185307179586476925286766559L;
      const long double part = turns - std::floor(turns);   // [0, 1)
      const long double scaled = std::floor(part * 18446744073709551616.0L + 0.5L);
      phases[i] = scaled >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(scaled);
    }
  });
}

int32_t sb_rotary(const sb_heads* x, const sb_heads* y, int32_t elem_type, int64_t tokens, int32_t heads, int32_t head_dim,
                  const void* positions, int32_t positions_int64, const sb_rotary_table* table, int32_t inverse,
                  void* stream) {
  return checked("sb_rotary", [&] {
    supported(elem_type == DT_FLOAT || elem_type == DT_FLOAT16 || elem_type == DT_BFLOAT16,
              std::string("element type ") + dtype_name(elem_type));
    need(tokens >= 0 && tokens <= kMostTokens && heads >= 0 && head_dim > 0 && heads < (1 << 20) && head_dim < (1 << 20),
         "sizes out of range");
    need(table != nullptr, "table is null");
    const k::RotaryView t = view(table, head_dim, inverse != 0);
    if (tokens == 0 || heads == 0) return;
    const size_t esz = dtype_size(elem_type);
    const k::HeadsView xv = view(x, "x", esz), yv = view(y, "y", esz);
    apart(yv, "y", tokens, heads, head_dim);
    need(positions != nullptr && aligned(positions, positions_int64 ? 8 : 4), "positions are null or misaligned");
    launched(k::rotary(xv, yv, elem_type, tokens, heads, head_dim, positions, positions_int64 ? 1 : 0, t,
                       multiprocessors(), static_cast<cudaStream_t>(stream)));
  });
}

int32_t sb_paged_append(const sb_paged_cache* cache, const sb_heads* k, const sb_heads* v, const sb_heads* q,
                        const sb_heads* q_out, int32_t q_heads, int64_t tokens, const int32_t* query_starts,
                        const sb_rotary_table* table, void* stream) {
  return checked("sb_paged_append", [&] {
    need((q == nullptr) == (q_out == nullptr), "q and q_out go together");
    need(q == nullptr || (table != nullptr && q_heads > 0), "q needs a table and q_heads");
    const k::PagedView c = view(cache, q ? q_heads : 0, tokens, query_starts);
    need(c.head_dim < (1 << 20) && c.kv_heads < (1 << 20) && c.q_heads < (1 << 20), "head sizes out of range");
    k::RotaryView t = {nullptr, 0, 0, 0, 1.f};
    if (table) t = view(table, c.head_dim, false);
    if (tokens == 0 || c.batch == 0) return;
    const k::HeadsView kv = view(k, "k", 2), vv = view(v, "v", 2);
    k::HeadsView qv = {nullptr, 0, 0}, ov = {nullptr, 0, 0};
    if (q) qv = view(q, "q", 2), ov = view(q_out, "q_out", 2), apart(ov, "q_out", tokens, q_heads, c.head_dim);
    launched(k::paged_append(c, cache->elem_type, kv, vv, qv, ov, t, multiprocessors(), static_cast<cudaStream_t>(stream)));
  });
}

int32_t sb_paged_attention_workspace(const sb_paged_cache* cache, int32_t q_heads, int64_t tokens, size_t* bytes) {
  return checked("sb_paged_attention_workspace", [&] {
    need(bytes != nullptr, "bytes is null");
    static const int32_t none = 0;   // the row starts do not matter to the size
    const k::PagedView c = view(cache, q_heads, tokens, &none);
    check_attention(c);
    *bytes = k::paged_attention_workspace(c, multiprocessors());
  });
}

int32_t sb_paged_attention(const sb_paged_cache* cache, const sb_heads* q, const sb_heads* out, int32_t q_heads,
                           int64_t tokens, const int32_t* query_starts, float scale, int32_t window, void* workspace,
                           size_t workspace_bytes, void* stream) {
  return checked("sb_paged_attention", [&] {
    const k::PagedView c = view(cache, q_heads, tokens, query_starts);
    check_attention(c);
    need(std::isfinite(scale) && scale > 0, "scale must be positive and finite");
    need(window >= 0, "window must not be negative");
    if (tokens == 0 || c.batch == 0) return;
    const k::HeadsView qv = view(q, "q", 2), ov = view(out, "out", 2);
    wide(qv, "q");
    wide(ov, "out");
    apart(ov, "out", tokens, q_heads, c.head_dim);
    wide({c.k, c.kt, c.kh}, "cache k");
    wide({c.v, c.vt, c.vh}, "cache v");
    supported(c.kp % 8 == 0 && c.vp % 8 == 0, "cache page strides need whole 8-element pieces");
    const int sms = multiprocessors();
    const size_t bytes = k::paged_attention_workspace(c, sms);
    need(workspace != nullptr && aligned(workspace, 256), "workspace is null or not 256-byte aligned");
    need(workspace_bytes >= bytes, "workspace has " + std::to_string(workspace_bytes) + " of " + std::to_string(bytes) + " bytes");
    launched(k::paged_attention(c, cache->elem_type, qv, ov, scale, window, workspace, sms, static_cast<cudaStream_t>(stream)));
  });
}

int32_t sb_decoder_status(void* stream) {
  return checked("sb_decoder_status", [&] {
    unsigned bits = 0;
    multiprocessors();   // a current device
    launched(k::paged_wait_errors(&bits, static_cast<cudaStream_t>(stream)));
    SB_CHECK(bits == 0, SB_CUDA_ERROR, "an attention kernel's pipeline wait timed out (code " + std::to_string(bits) + ")");
  });
}

int32_t sb_w4_layout_bytes(const sb_w4_weights* weights, size_t* bytes) {
  return checked("sb_w4_layout_bytes", [&] {
    need(bytes != nullptr, "bytes is null");
    *bytes = k::w4_layout_bytes(view(weights));
  });
}

int32_t sb_w4_layout(const sb_w4_weights* weights, const uint8_t* packed, int64_t packed_row_bytes, const void* scales,
                     const uint8_t* zeros, void* data, void* stream) {
  return checked("sb_w4_layout", [&] {
    const k::W4View w = view(weights);
    need(packed != nullptr && scales != nullptr && data != nullptr, "null buffer");
    need(aligned(scales, 2) && aligned(data, 256), "scales or data is misaligned");
    need((zeros != nullptr) == (w.zeros != 0), "zeros and has_zeros go together");
    need(packed_row_bytes >= (w.k + 1) / 2 && packed_row_bytes < kMostStride, "packed_row_bytes is shorter than a row");
    launched(k::w4_layout(w, packed, packed_row_bytes, scales, zeros, data, static_cast<cudaStream_t>(stream)));
  });
}

int32_t sb_linear_w4(const sb_w4_weights* weights, const void* x, int64_t x_row_stride, const void* bias, void* y,
                     int64_t y_row_stride, int64_t rows, void* stream) {
  return checked("sb_linear_w4", [&] {
    const k::W4View w = view(weights);
    need(rows >= 0 && rows <= kMostTokens, "rows out of range");
    if (rows == 0) return;
    need(w.data != nullptr && aligned(w.data, 256), "weights data is null or misaligned");
    need(x != nullptr && y != nullptr && aligned(x, 2) && aligned(y, 2) && aligned(bias, 2), "x, y or bias is null or misaligned");
    need(usable(x_row_stride) && usable(y_row_stride), "row stride out of range");
    need(rows == 1 || std::llabs(y_row_stride) >= w.n, "rows of y overlap");
    launched(k::linear_w4(w, x, x_row_stride, bias, y, y_row_stride, rows, multiprocessors(), static_cast<cudaStream_t>(stream)));
  });
}

}  // extern "C"
