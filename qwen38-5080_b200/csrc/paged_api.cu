// C-ABI of the paged FP8 cache: argument checks on the host, then launches on the caller's stream.  Nothing here
// allocates, synchronises or reads device memory.
#include "paged.cuh"

using namespace b200attn;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int resolve_paged(const B200AttnPagedShape* s, PagedGeometry* g) {
  if (!s) return B200ATTN_ERR_NULL;
  if (s->n_layers < 1 || s->batch < 1 || s->h_q < 1 || s->h_kv < 1 || s->n_pages < 1 || s->max_pages < 1) return B200ATTN_ERR_SHAPE;
  if (s->head_dim != 128 && s->head_dim != 256) return B200ATTN_ERR_SHAPE;
  if (s->page_size != 16 && s->page_size != 32 && s->page_size != 64 && s->page_size != 128) return B200ATTN_ERR_SHAPE;
  if (s->h_q % s->h_kv || s->h_q / s->h_kv > kMaxGroup) return B200ATTN_ERR_SHAPE;
  if (s->reserved != 0 || s->reserved2 != 0) return B200ATTN_ERR_SHAPE;
  if ((long long)s->n_layers * s->batch > 65535) return B200ATTN_ERR_SHAPE;
  // token slots are 32-bit, and so are the token rows of one layer (copy coordinates)
  if ((long long)s->max_pages * s->page_size > 0x7fffffffLL - 256) return B200ATTN_ERR_SHAPE;
  if ((long long)s->n_pages * s->h_kv * s->page_size > 0x7fffffffLL) return B200ATTN_ERR_SHAPE;
  const long long dense = (long long)s->n_pages * s->h_kv * s->page_size * s->head_dim;
  g->n_layers = s->n_layers; g->batch = s->batch; g->h_q = s->h_q; g->h_kv = s->h_kv; g->head_dim = s->head_dim;
  g->page_size = s->page_size; g->n_pages = s->n_pages; g->max_pages = s->max_pages; g->group = s->h_q / s->h_kv;
  g->k_layer_stride = s->k_layer_stride ? s->k_layer_stride : dense;
  g->v_layer_stride = s->v_layer_stride ? s->v_layer_stride : dense;
  if (s->n_layers > 1 && (g->k_layer_stride < dense || g->v_layer_stride < dense)) return B200ATTN_ERR_SHAPE;
  if ((g->k_layer_stride & 15) || (g->v_layer_stride & 15)) return B200ATTN_ERR_ALIGN;
  return B200ATTN_OK;
}

int check_rope(const B200AttnRope* r, const PagedGeometry& g) {
  if (r->reserved != 0) return B200ATTN_ERR_SHAPE;
  if (!r->cos || !r->sin) return B200ATTN_ERR_NULL;
  if (r->rotary_dim < 16 || r->rotary_dim > g.head_dim || r->rotary_dim % 16) return B200ATTN_ERR_SHAPE;
  if (r->n_positions < 1 || r->n_axes < 1 || r->n_axes > 4 || (!r->positions && r->n_axes != 1)) return B200ATTN_ERR_SHAPE;
  if (!aligned16(r->cos) || !aligned16(r->sin) || !aligned16(r->pair_axis)) return B200ATTN_ERR_ALIGN;
  return B200ATTN_OK;
}

}  // namespace

extern "C" {

int b200attn_paged_rope_append(const B200AttnPagedShape* shape, const B200AttnRope* rope, int n_tokens, const int* q_start,
                               const void* q, const void* k, const void* v, const void* q_norm_weight, const void* k_norm_weight,
                               float eps, void* q_out, void* k_pages, void* v_pages, float* k_scale, float* v_scale,
                               const int* page_table, int* seq_pos, int advance_pos, int* status, void* stream) {
  PagedGeometry g;
  int rc = resolve_paged(shape, &g);
  if (rc) return rc;
  if (!k || !v || !k_pages || !v_pages || !k_scale || !v_scale || !page_table || !seq_pos || !status) return B200ATTN_ERR_NULL;
  if ((q == nullptr) != (q_out == nullptr)) return B200ATTN_ERR_NULL;
  if (n_tokens < 0 || (!q_start && n_tokens != g.batch)) return B200ATTN_ERR_SHAPE;
  if (!(eps >= 0.f)) return B200ATTN_ERR_SHAPE;
  if (rope && (rc = check_rope(rope, g))) return rc;
  if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(q_norm_weight) || !aligned16(k_norm_weight))
    return B200ATTN_ERR_ALIGN;
  const PagedAppendArgs a{rope, n_tokens, q_start, q, k, v, q_norm_weight, k_norm_weight, eps, q_out, k_pages, v_pages,
                          k_scale, v_scale, page_table, seq_pos, advance_pos, status};
  const cudaError_t e = launch_paged_append(g, a, (cudaStream_t)stream);
  return e == cudaSuccess ? B200ATTN_OK : record_cuda_error(e);
}

int b200attn_paged_workspace_bytes(const B200AttnPagedShape* shape, int q_tokens, int max_seq_len, size_t* bytes) {
  PagedGeometry g;
  int rc = resolve_paged(shape, &g);
  if (rc) return rc;
  if (!bytes) return B200ATTN_ERR_NULL;
  if (q_tokens < 0) return B200ATTN_ERR_SHAPE;
  if (max_seq_len < 0) return B200ATTN_ERR_CAPACITY;
  *bytes = q_tokens ? paged_prefill_workspace_bytes(g) : paged_decode_workspace_bytes();
  return B200ATTN_OK;
}

static int check_attention(const B200AttnPagedShape* shape, PagedGeometry* g, const PagedAttnArgs& a, bool prefill) {
  int rc = resolve_paged(shape, g);
  if (rc) return rc;
  if (!a.q || !a.k_pages || !a.v_pages || !a.k_scale || !a.v_scale || !a.page_table || !a.seq_len || !a.out || !a.status) return B200ATTN_ERR_NULL;
  if (prefill && !a.q_start) return B200ATTN_ERR_NULL;
  if (a.n_tokens < 0) return B200ATTN_ERR_SHAPE;
  if (!(a.softmax_scale >= 0.f && a.softmax_scale <= 3.402823466e38f)) return B200ATTN_ERR_SHAPE;   // the kernels count on multipliers >= 0
  if (a.max_seq_len < 0) return B200ATTN_ERR_CAPACITY;
  if (!aligned16(a.q) || !aligned16(a.k_pages) || !aligned16(a.v_pages) || !aligned16(a.out) || !aligned16(a.workspace)) return B200ATTN_ERR_ALIGN;
  const size_t need = prefill ? paged_prefill_workspace_bytes(*g) : paged_decode_workspace_bytes();
  if (need && !a.workspace) return B200ATTN_ERR_NULL;
  if (a.workspace_bytes < need) return B200ATTN_ERR_WORKSPACE;
  return B200ATTN_OK;
}

int b200attn_paged_decode(const B200AttnPagedShape* shape, const void* q, const void* k_pages, const void* v_pages,
                          const float* k_scale, const float* v_scale, const int* page_table, const int* seq_len, int seq_len_offset,
                          int max_seq_len, float softmax_scale, void* workspace, size_t workspace_bytes, void* out, int* status,
                          void* stream) {
  PagedGeometry g;
  const PagedAttnArgs a{q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, seq_len_offset, max_seq_len, softmax_scale,
                        workspace, workspace_bytes, out, status, 0, nullptr, 0};
  const int rc = check_attention(shape, &g, a, false);
  if (rc) return rc;
  const cudaError_t e = launch_paged_decode(g, a, (cudaStream_t)stream);
  return e == cudaSuccess ? B200ATTN_OK : record_cuda_error(e);
}

int b200attn_paged_prefill(const B200AttnPagedShape* shape, int n_tokens, const void* q, const int* q_start, const void* k_pages,
                           const void* v_pages, const float* k_scale, const float* v_scale, const int* page_table, const int* seq_len,
                           int max_seq_len, int causal, float softmax_scale, void* workspace, size_t workspace_bytes, void* out,
                           int* status, void* stream) {
  PagedGeometry g;
  const PagedAttnArgs a{q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, 0, max_seq_len, softmax_scale,
                        workspace, workspace_bytes, out, status, n_tokens, q_start, causal};
  const int rc = check_attention(shape, &g, a, true);
  if (rc) return rc;
  if (n_tokens == 0) return B200ATTN_OK;
  const cudaError_t e = launch_paged_prefill(g, a, (cudaStream_t)stream);
  return e == cudaSuccess ? B200ATTN_OK : record_cuda_error(e);
}

}  // extern "C"
