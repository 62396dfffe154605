// The paged FP8 cache: resolved geometry, launch arguments and the small device helpers its kernels share.
#pragma once

#include "common.cuh"

namespace b200attn {

struct PagedGeometry {
  int n_layers, batch, h_q, h_kv, head_dim, page_size, n_pages, max_pages, group;
  long long k_layer_stride, v_layer_stride;   // bytes, always filled in
};

struct PagedAppendArgs {
  const B200AttnRope* rope;   // null = no rotation
  int n_tokens;
  const int* q_start;         // null = one token per sequence
  const void *q, *k, *v, *wq, *wk;
  float eps;
  void* q_out;
  void *k_pages, *v_pages;
  float *k_scale, *v_scale;
  const int* page_table;
  int* seq_pos;
  int advance_pos;
  int* status;
};
cudaError_t launch_paged_append(const PagedGeometry& g, const PagedAppendArgs& a, cudaStream_t stream);

struct PagedAttnArgs {
  const void* q;
  const void *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int *page_table, *seq_len;
  int seq_len_offset, max_seq_len;
  float softmax_scale;
  void* workspace;
  size_t workspace_bytes;
  void* out;
  int* status;
  // many query tokens per sequence
  int n_tokens;
  const int* q_start;
  int causal;
};
size_t paged_decode_workspace_bytes();
cudaError_t launch_paged_decode(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream);
size_t paged_prefill_workspace_bytes(const PagedGeometry& g);
cudaError_t launch_paged_prefill(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream);
bool few_rows(const PagedGeometry& g, int n_tokens);
size_t paged_few_partial_bytes(const PagedGeometry& g);
cudaError_t launch_paged_few(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream);

// A workspace: counters (zero between launches; a call that joins pieces has at most three tiles per SM to join), the stream-K
// kernel's tagged words (zero between launches), partial results (anything).  The parts begin at the same place for every kernel
// and shape, so calls that do not overlap in time may share a workspace whatever they are.
constexpr size_t kPagedWordBytes = 8 * 2 * (8 * 128 + 16);   // per CTA: two states of 8 heads of 128 (of 256: one CTA per SM, not three)
inline size_t paged_words_offset() { return ((size_t)device_sms() * 12 + 255) & ~(size_t)255; }
inline size_t paged_partials_offset() { return paged_words_offset() + 3 * (size_t)device_sms() * kPagedWordBytes; }
inline int* paged_counters(void* ws) { return (int*)ws; }
inline unsigned long long* paged_words(void* ws) { return (unsigned long long*)((uint8_t*)ws + paged_words_offset()); }
inline float* paged_partials(void* ws) { return (float*)((uint8_t*)ws + paged_partials_offset()); }

// The least scale that V is held relative to where that is the largest of the keys so far: its reciprocal is finite, that of a
// subnormal scale may not be.
constexpr float kLeastScale = 0x1p-126f;

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ unsigned long long pair2(float x, float y) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void split2(unsigned long long p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Plain loads, not the non-coherent ones: a dependent launch can begin while the kernel that writes the data still runs (it reads them
// after its wait), and non-coherent loads are for data that nobody writes during the kernel.
template <class T>
__device__ __forceinline__ T ld(const T* p) { return *p; }

// For the index checks: whether token rows [row, row + n) of a layer's pool exist.
__device__ __forceinline__ bool rows_exist(const PagedGeometry& g, long long row, int n, int layer) {
  return row >= 0 && row + n <= (long long)g.n_pages * g.h_kv * g.page_size && layer >= 0 && layer < g.n_layers;
}

// Whether sequence b of a packed call may own tokens [q0, end).
__device__ __forceinline__ bool range_fits(int q0, int end, int n_tokens, int* status, bool report) {
  const bool fits = q0 >= 0 && end >= q0 && end <= n_tokens;
  if (!fits && report) atomicOr(status, B200ATTN_STATUS_BAD_RANGE);
  return fits;
}

// Valid length of a sequence: negative lengths count as 0, lengths beyond the table's capacity are clamped to it.
__device__ __forceinline__ int paged_len(const PagedGeometry& g, long long raw, int* status, bool report) {
  const long long cap = (long long)g.max_pages * g.page_size;
  if (raw < 0) {
    if (report) atomicOr(status, B200ATTN_STATUS_LEN_NEGATIVE);
    return 0;
  }
  if (raw > cap) {
    if (report) atomicOr(status, B200ATTN_STATUS_LEN_OVER_CAP);
    return (int)cap;
  }
  return (int)raw;
}

}  // namespace b200attn
