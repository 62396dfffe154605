// Attention over the paged FP8 cache, the plain way: one warp per query row and head, one key at a time, running
// maximum and sum in fp32.
#include "paged.cuh"

namespace b200attn {

namespace {

struct SimpleParams {
  PagedGeometry g;
  const uint16_t* q;
  const uint8_t *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int *page_table, *seq_len, *q_start;
  int seq_len_offset, n_tokens, causal;
  float scale;
  uint16_t* out;
  int* status;
};

template <int D>
__global__ void __launch_bounds__(256) paged_simple_kernel(const SimpleParams p) {
  constexpr int E = D / 32;
  const PagedGeometry& g = p.g;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (long long)g.n_layers * p.n_tokens * g.h_q) return;
  const int hq = (int)(w % g.h_q), h = hq / g.group;
  const long long lt = w / g.h_q;
  const int token = (int)(lt % p.n_tokens), layer = (int)(lt / p.n_tokens);
  int b = token, len;
  if (p.q_start) {
    if (token < p.q_start[0] || token >= p.q_start[g.batch]) return;
    int lo = 0, hi = g.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.q_start[mid] <= token) lo = mid; else hi = mid - 1;
    }
    b = lo;
    len = paged_len(g, p.seq_len[b], p.status, lane == 0);
    if (p.causal) len = min(len, max(0, len - (p.q_start[b + 1] - token) + 1));
  } else {
    len = paged_len(g, p.seq_len[b] + p.seq_len_offset, p.status, lane == 0);
  }
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = bf16_bits_to_float(p.q[w * D + lane * E + e]) * p.scale;
    acc[e] = 0.f;
  }
  for (int t = 0; t < len; ++t) {
    const int page = p.page_table[(long long)b * g.max_pages + t / g.page_size];
    if (page < 0 || page >= g.n_pages) {
      if (lane == 0) atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE);
      continue;
    }
    const long long si = ((long long)layer * g.n_pages + page) * g.h_kv + h;
    const long long off = (((long long)page * g.h_kv + h) * g.page_size + t % g.page_size) * D + lane * E;
    const uint8_t* kp = p.k_pages + layer * g.k_layer_stride + off;
    const uint8_t* vp = p.v_pages + layer * g.v_layer_stride + off;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 f = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(kp + e));
      s += q[e] * f.x + q[e + 1] * f.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.k_scale[si];
    const float mn = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - mn), pr = expf(s - mn) ;
    m = mn;
    l = l * keep + pr;
    const float pv = pr * p.v_scale[si];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 f = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(vp + e));
      acc[e] = acc[e] * keep + pv * f.x;
      acc[e + 1] = acc[e + 1] * keep + pv * f.y;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const __nv_bfloat16 o = __float2bfloat16_rn(acc[e] * inv);
    p.out[w * D + lane * E + e] = *reinterpret_cast<const uint16_t*>(&o);
  }
}

cudaError_t launch_simple(const PagedGeometry& g, const PagedAttnArgs& a, int n_tokens, const int* q_start, cudaStream_t stream) {
  SimpleParams p{g, (const uint16_t*)a.q, (const uint8_t*)a.k_pages, (const uint8_t*)a.v_pages, a.k_scale, a.v_scale,
                 a.page_table, a.seq_len, q_start, a.seq_len_offset, n_tokens, a.causal, a.softmax_scale, (uint16_t*)a.out, a.status};
  const long long grid = ((long long)g.n_layers * n_tokens * g.h_q + 7) / 8;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (grid == 0) return cudaSuccess;
  if (g.head_dim == 128) paged_simple_kernel<128><<<(unsigned)grid, 256, 0, stream>>>(p);
  else paged_simple_kernel<256><<<(unsigned)grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t paged_prefill_workspace_bytes(const PagedGeometry&, int, int) { return 0; }
cudaError_t launch_paged_prefill(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  return launch_simple(g, a, a.n_tokens, a.q_start, stream);
}

}  // namespace b200attn
