// Host-side launchers of the kernels for positions and generation: rotation by positions, a paged key / value cache in
// 8 bits, sampling.  Plain CUDA types only; dtype codes as in kernels.h.  Launchers return 0, or why they refuse.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace slapo {

// Positions of tokens: start + s, from memory (32 or 64 bits wide) where `ids` is set, or those of a cache's new tokens
// where `lengths` is: the first counts[b] (or all) of S end at lengths[b], others have none
struct RotaryPositions {
  const void* ids;
  bool ids64;
  int64_t batch_stride, token_stride;      // elements
  int64_t start;
  const int32_t *lengths, *counts;
};
// Heads [B, S, heads, D] that are turned, or copied, from x to y; strides in elements, D contiguous
struct RotaryPart {
  const void* x;
  void* y;
  int64_t x_stride[3], y_stride[3];
  int heads;
  bool turn;
};
struct RotaryCall {
  RotaryPart part[3];
  int parts;
  const float* table;       // [rows, rotary / 2, 2]: cosine, sine
  int64_t table_rows;
  RotaryPositions at;
  int64_t B, S;
  int D, rotary;            // rotary 0: heads are copied, zeros where a position is none
  bool interleaved, transposed;      // transposed: the gradient's direction
  bool beside;                       // the kernel launched before may still run, and says when this one may begin
  int dtype;
};
int launch_rotary(const RotaryCall& c, cudaStream_t stream);

// A cache of pages [n_pages, 2, heads, page, pitch] of e4m3 numbers with their scales [n_pages, 2, heads], and the
// sequences in it: `table` [B, table_pages] names their pages, `lengths` [B] counts their tokens, new ones among them,
// `counts` [B] (or null: all n) how many of the n new ones they bring.
struct PagedCache {
  uint8_t* pages;
  float* scales;
  int64_t n_pages;
  int heads, page, dim, pitch;
  const int32_t* table;
  int table_pages;
  const int32_t* lengths;
  const int32_t* counts;
  int B, n;
};
struct PagedAppend {
  PagedCache cache;
  const void *k, *v, *q;      // [B, n, heads, D]; q, with heads of its own: or null
  void* q_out;                // [B, n, q_heads, D]
  int64_t k_stride[3], v_stride[3], q_stride[3];
  int q_heads;
  const float* rot;           // rotation's table [rot_rows, rotary / 2, 2], or null
  int64_t rot_rows;
  int rotary;
  bool interleaved;
  int dtype;
};
int launch_paged_append(const PagedAppend& c, cudaStream_t stream);

struct PagedAttention {
  PagedCache cache;
  const void* q;              // [B, n, q_heads, D]
  int64_t q_stride[3];
  int q_heads;
  void* out;                  // [B, n, q_heads, D]
  float scale;
  int window;                 // 0: all keys
  bool bf16;
  float* scratch;             // paged_attention_words() floats
};
int64_t paged_attention_words(const PagedAttention& c);
int launch_paged_attention(const PagedAttention& c, cudaStream_t stream);

// A setting that is one number or one for each row
template <typename T>
struct PerRow {
  const T* rows;
  T value;
};
struct SampleCall {
  const void* logits;
  int64_t row_stride;
  const float* uniform;
  PerRow<float> temperature, top_p, min_p;
  PerRow<int> top_k;
  int64_t* out;
  int64_t rows;
  int vocab;
  int dtype;
};
constexpr int kSampleVocab = 1 << 18;
int launch_sample(const SampleCall& c, cudaStream_t stream);

#ifdef __CUDACC__
// x c + y s, the same to the bit in every kernel and form (a compiler may contract either product)
__device__ __forceinline__ float turned_value(float x, float c, float y, float s) {
  return __fmaf_rn(x, c, __fmul_rn(y, s));
}
#endif

}  // namespace slapo
