// Append to the paged FP8 cache: optional RMS norm of the query and key heads, rotary embedding (positions on one to
// four axes), and quantise-and-append of the key and the value with one power-of-two scale per (layer, page, kv head).
//
//   y = x * rsqrt(mean(x^2) + eps) * (1 + w)                                   (query and key, if a weight is given)
//   r_j = y_j cos - y_{j+R/2} sin,  r_{j+R/2} = y_{j+R/2} cos + y_j sin        (j < R/2, angle of pos[axis(j)])
//   s   = 2^ceil(log2(max |r| / 448)) over the new tokens of the page; max(that, old scale) if the page held tokens
//   byte = e4m3(r / s);  earlier rows, if the scale grew: byte = e4m3(value(byte) * old / s)
//
// Why a power of two: the page's scale is not known before its last token has come, so it has to be able to grow,
// and a growing scale re-expresses the earlier rows.  With powers of two that is a change of exponent, exact unless a
// value becomes subnormal, however often it happens; with amax / 448 every growth would round all earlier rows again.
// e4m3 keeps its 4 significant bits over 15 binades, so the binade that rounding the scale up can cost is not felt.
//
// Bound: HBM bytes (query in and out, key and value in, bytes out), and for single tokens the launch.
#include "paged.cuh"

namespace b200attn {

namespace {

struct AppendParams {
  PagedGeometry g;
  int n_tokens;
  const int* q_start;
  const uint16_t *q, *k, *v, *wq, *wk;
  float eps;
  uint16_t* q_out;
  uint8_t *k_pages, *v_pages;
  float *k_scale, *v_scale;
  const int* page_table;
  const int* seq_pos;
  int* status;
  const float *cos, *sin;
  const int *positions, *pair_axis;
  int n_positions, n_axes, rot;
  int kv_blocks;
};

// Smallest power of two s with amax / s <= 448 = 1.75 * 2^8, at least 2^-126; amax is finite and >= 0.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // biased exponent of s
  return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;   // NaN and infinities do not take part in the maximum
}

// 8 bf16 -> floats
__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// 8 floats -> 8 e4m3 bytes: nearest even, saturating at 448; NaN -> 0x7F
__device__ __forceinline__ uint2 quant8(const float (&x)[8], float inv) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x[2 * i + 1] * inv), "f"(x[2 * i] * inv));
    h[i] = r;
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
// 16 e4m3 bytes re-expressed in a larger power-of-two scale: value * ratio, ratio = old / new < 1
__device__ __forceinline__ uint4 rescale16(const uint4& raw, float ratio) {
  float f[16];
  e4m3x16_to_float(raw, f);
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { a[i] = f[i]; b[i] = f[8 + i]; }
  const uint2 lo = quant8(a, ratio), hi = quant8(b, ratio);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// What a lane needs to rotate its 8 dims of a head: cosines, sines (0 / identity beyond rot) for one token.
template <int D>
struct Rotation {
  static constexpr int TPR = D / 8;   // lanes per head row
  float c[8], s[8];
  int partner;                        // lane that holds the other half of the pairs
  bool on, low;

  __device__ __forceinline__ void load(const AppendParams& p, int lane, int token, int slot) {
    const int lr = lane % TPR, i0 = lr * 8, half = p.rot >> 1;
    on = i0 < p.rot;
    low = i0 < half;
    partner = lane + (on ? (low ? half / 8 : -(half / 8)) : 0);
    if (!on) return;
    const int j0 = low ? i0 : i0 - half;
    if (p.pair_axis == nullptr) {
      int pos = p.positions ? p.positions[token] : slot;
      if (pos < 0 || pos >= p.n_positions) {
        atomicOr(p.status, B200ATTN_STATUS_BAD_POSITION);
        pos = pos < 0 ? 0 : p.n_positions - 1;
      }
      const float4* cp = reinterpret_cast<const float4*>(p.cos + (long long)pos * half + j0);
      const float4* sp = reinterpret_cast<const float4*>(p.sin + (long long)pos * half + j0);
      const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
      c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
      s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int ax = __ldg(p.pair_axis + j0 + e);
        bool bad = ax < 0 || ax >= p.n_axes;
        ax = bad ? 0 : ax;
        int pos = p.positions ? p.positions[(long long)ax * p.n_tokens + token] : slot;
        bad |= pos < 0 || pos >= p.n_positions;
        if (bad) atomicOr(p.status, B200ATTN_STATUS_BAD_POSITION);
        pos = pos < 0 ? 0 : (pos >= p.n_positions ? p.n_positions - 1 : pos);
        c[e] = __ldg(p.cos + (long long)pos * half + j0 + e);
        s[e] = __ldg(p.sin + (long long)pos * half + j0 + e);
      }
    }
  }
  // Every lane of the warp calls it (lanes of absent rows with zeros).
  __device__ __forceinline__ void turn(float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl_sync(0xffffffffu, x[e], partner & 31);
      if (on) x[e] = low ? x[e] * c[e] - other * s[e] : x[e] * c[e] + other * s[e];
    }
  }
};

// RMS norm over the head's TPR lanes; every lane of the warp calls it.
template <int D>
__device__ __forceinline__ void rms_norm(float (&x)[8], const float (&w1)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
  for (int off = D / 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  const float inv = __frsqrt_rn(ss * (1.f / D) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w1[e];
}
template <int D>
__device__ __forceinline__ void load_norm(const uint16_t* w, int layer, int lane, float (&w1)[8]) {
  float t[8];
  unpack8(__ldg(reinterpret_cast<const uint4*>(w + (long long)layer * D) + lane % (D / 8)), t);
#pragma unroll
  for (int e = 0; e < 8; ++e) w1[e] = 1.f + t[e];
}

// Sequence that owns packed token t (largest b with q_start[b] <= t; empty sequences share their start).
__device__ __forceinline__ int sequence_of(const int* q_start, int batch, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (q_start[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int page_of(const AppendParams& p, int b, int page_index) {
  const int id = p.page_table[(long long)b * p.g.max_pages + page_index];
  return id >= 0 && id < p.g.n_pages ? id : -1;
}

// Query rows: one warp per token, its heads in turn; the rotation is loaded once per token.
template <int D>
__device__ __forceinline__ void rotate_queries(const AppendParams& p, long long first_warp, long long n_warps) {
  constexpr int TPR = D / 8, RPW = 32 / TPR;   // head rows per warp step
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)p.g.n_layers * p.n_tokens;
  for (long long r = first_warp; r < rows; r += n_warps) {
    const int layer = (int)(r / p.n_tokens), token = (int)(r % p.n_tokens);
    int b = token, slot;
    if (p.q_start) {
      if (token >= p.q_start[p.g.batch] || token < p.q_start[0]) continue;   // a row that belongs to nobody
      b = sequence_of(p.q_start, p.g.batch, token);
      slot = p.seq_pos[b] + token - p.q_start[b];
    } else {
      slot = p.seq_pos[b];
    }
    Rotation<D> rot;
    rot.load(p, lane, token, slot);
    float w1[8];
    if (p.wq) load_norm<D>(p.wq, layer, lane, w1);
    const uint4* src = reinterpret_cast<const uint4*>(p.q) + r * p.g.h_q * TPR;
    uint4* dst = reinterpret_cast<uint4*>(p.q_out) + r * p.g.h_q * TPR;
    for (int h0 = 0; h0 < p.g.h_q; h0 += RPW) {
      const int h = h0 + lane / TPR;
      float x[8] = {};
      if (h < p.g.h_q) unpack8(src[h * TPR + lane % TPR], x);
      if (p.wq) rms_norm<D>(x, w1, p.eps);
      rot.turn(x);
      if (h < p.g.h_q) dst[h * TPR + lane % TPR] = pack8(x);
    }
  }
}

// One token per sequence.  One warp per key or value row (its first TPR lanes hold the row; all 32 re-express the page's
// earlier rows when the scale grows), the warps behind them rotate the queries.
template <int D>
__global__ void __launch_bounds__(256)
paged_append_token_kernel(const AppendParams p) {
  constexpr int TPR = D / 8;
  const PagedGeometry& g = p.g;
  const int lane = threadIdx.x & 31;
  const long long warp = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long kv_rows = (long long)g.n_layers * g.batch * g.h_kv * 2;
  if (warp >= kv_rows) {
    if (p.q) rotate_queries<D>(p, warp - kv_rows, (long long)gridDim.x * 8 - kv_rows);
    return;
  }
  const int which = (int)(warp & 1);                 // 0 key, 1 value
  const long long row = warp >> 1;                   // (layer, sequence, head)
  const int h = (int)(row % g.h_kv);
  const long long lb = row / g.h_kv;
  const int b = (int)(lb % g.batch), layer = (int)(lb / g.batch);
  const int pos = p.seq_pos[b];
  if (pos < 0 || pos >= (long long)g.max_pages * g.page_size) {
    if (lane == 0) atomicOr(p.status, B200ATTN_STATUS_POS_AT_CAPACITY);
    return;
  }
  const int fill = pos % g.page_size, page = page_of(p, b, pos / g.page_size);
  if (page < 0) {
    if (lane == 0) atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE);
    return;
  }
  float x[8] = {};
  if (lane < TPR) unpack8(reinterpret_cast<const uint4*>(which ? p.v : p.k)[row * TPR + lane], x);
  if (!which) {
    if (p.wk) {
      float w1[8];
      load_norm<D>(p.wk, layer, lane, w1);
      rms_norm<D>(x, w1, p.eps);
    }
    Rotation<D> rot;
    rot.load(p, lane, b, pos);
    rot.turn(x);
  }
  float amax = 0.f;
  if (lane < TPR)
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(x[e]));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  float s = pow2_scale(amax);
  float* sp = (which ? p.v_scale : p.k_scale) + ((long long)layer * g.n_pages + page) * g.h_kv + h;
  uint8_t* base = (which ? p.v_pages : p.k_pages) + (long long)layer * (which ? g.v_layer_stride : g.k_layer_stride) +
                  ((long long)page * g.h_kv + h) * g.page_size * D;
  if (fill > 0) {
    const float old = *sp;
    if (s > old) {
      const float ratio = old / s;
      uint4* rows16 = reinterpret_cast<uint4*>(base);
      const int n = fill * (D / 16);
#pragma unroll 4
      for (int i = lane; i < n; i += 32) rows16[i] = rescale16(rows16[i], ratio);
    } else {
      s = old;
    }
  }
  __syncwarp();
  if (lane == 0) *sp = s;
  if (lane < TPR) reinterpret_cast<uint2*>(base + (long long)fill * D)[lane] = quant8(x, __fdiv_rn(1.f, s));
}

// Prompts.  A thread block holds the new tokens of one (layer, page, kv head) of keys or of values: rotates them, finds
// their scale, writes them.  The blocks behind those rotate the queries.  NP: passes of THREADS / TPR rows over a page.
template <int D, int NP, int THREADS>
__global__ void __launch_bounds__(THREADS)
paged_append_prompt_kernel(const AppendParams p) {
  constexpr int TPR = D / 8, RPP = THREADS / TPR;
  const PagedGeometry& g = p.g;
  const int tid = threadIdx.x, lane = tid & 31;
  const long long units = (long long)p.kv_blocks * g.h_kv * 2 * g.n_layers;
  if (blockIdx.x >= units) {
    if (p.q) rotate_queries<D>(p, ((long long)blockIdx.x - units) * (THREADS / 32) + (tid >> 5), ((long long)gridDim.x - units) * (THREADS / 32));
    return;
  }
  const int which = (int)(blockIdx.x & 1);
  long long u = blockIdx.x >> 1;
  const int h = (int)(u % g.h_kv);
  u /= g.h_kv;
  const int chunk = (int)(u % p.kv_blocks), layer = (int)(u / p.kv_blocks);

  // the sequence and page that chunk number `chunk` of the call is: a scan over the sequences' touched pages
  __shared__ int s_seq, s_page;
  __shared__ float s_max[THREADS / 32];
  if (tid < 32) {
    int before = 0;
    if (tid == 0) s_seq = -1;
    __syncwarp();
    for (int b0 = 0; b0 < g.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0, first = 0;
      if (b < g.batch) {
        const int q0 = p.q_start[b], nt = p.q_start[b + 1] - q0, pos = p.seq_pos[b];
        if (nt > 0 && pos >= 0 && q0 >= 0 && q0 + nt <= p.n_tokens) {
          first = pos / g.page_size;
          n = (int)(((long long)pos + nt - 1) / g.page_size) - first + 1;
        }
      }
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += t;
      }
      const int start = before + inc - n;
      if (n > 0 && chunk >= start && chunk < start + n) { s_seq = b; s_page = first + chunk - start; }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > chunk) break;
    }
  }
  __syncthreads();
  const int b = s_seq;
  if (b < 0) return;                                     // the grid is an upper bound
  const int page_index = s_page;
  const int q0 = p.q_start[b], nt = p.q_start[b + 1] - q0, pos = p.seq_pos[b];
  const int page = page_index < g.max_pages ? page_of(p, b, page_index) : -1;
  if (page < 0) {
    if (tid == 0) atomicOr(p.status, page_index < g.max_pages ? B200ATTN_STATUS_BAD_PAGE : B200ATTN_STATUS_POS_AT_CAPACITY);
    return;
  }
  const int slot0 = page_index * g.page_size;
  const int lo = max(pos - slot0, 0);                                                   // rows [lo, hi) are new
  const int hi = (int)min((long long)g.page_size, (long long)pos + nt - slot0);

  float x[NP][8];
  float w1[8];
  const bool norm = !which && p.wk != nullptr;
  if (norm) load_norm<D>(p.wk, layer, lane, w1);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = i * RPP + tid / TPR;
    const bool mine = row >= lo && row < hi;
    const int token = q0 + slot0 + row - pos;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
    if (mine)
      unpack8(reinterpret_cast<const uint4*>(which ? p.v : p.k)[(((long long)layer * p.n_tokens + token) * g.h_kv + h) * TPR + tid % TPR], x[i]);
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = i * RPP + tid / TPR;
    const bool mine = row >= lo && row < hi;
    if (!which) {
      if (norm) rms_norm<D>(x[i], w1, p.eps);
      Rotation<D> rot;
      const int safe = min(max(row, lo), hi - 1);
      rot.load(p, lane, q0 + slot0 + safe - pos, slot0 + safe);
      rot.turn(x[i]);
    }
    if (mine)
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(x[i][e]));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if (lane == 0) s_max[tid >> 5] = amax;
  float* sp = (which ? p.v_scale : p.k_scale) + ((long long)layer * g.n_pages + page) * g.h_kv + h;
  const float old = lo > 0 ? *sp : 0.f;
  __syncthreads();                                        // maxima are in; every thread has read the old scale
  amax = s_max[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) amax = fmaxf(amax, s_max[i]);
  float s = pow2_scale(amax);
  uint8_t* base = (which ? p.v_pages : p.k_pages) + (long long)layer * (which ? g.v_layer_stride : g.k_layer_stride) +
                  ((long long)page * g.h_kv + h) * g.page_size * D;
  if (lo > 0) {
    if (s > old) {
      const float ratio = old / s;
      uint4* rows16 = reinterpret_cast<uint4*>(base);
      for (int i = tid; i < lo * (D / 16); i += THREADS) rows16[i] = rescale16(rows16[i], ratio);
    } else {
      s = old;
    }
  }
  if (tid == 0) *sp = s;
  const float inv = __fdiv_rn(1.f, s);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = i * RPP + tid / TPR;
    if (row >= lo && row < hi) reinterpret_cast<uint2*>(base + (long long)row * D)[tid % TPR] = quant8(x[i], inv);
  }
}

__global__ void paged_advance_kernel(PagedGeometry g, const int* q_start, int* seq_pos) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= g.batch) return;
  const int n = q_start ? q_start[b + 1] - q_start[b] : 1, p = seq_pos[b];
  if (p >= 0 && n >= 0 && (long long)p + n <= (long long)g.max_pages * g.page_size) seq_pos[b] = p + n;
}

}  // namespace

cudaError_t launch_paged_append(const PagedGeometry& g, const PagedAppendArgs& a, cudaStream_t stream) {
  AppendParams p{};
  p.g = g;
  p.n_tokens = a.n_tokens;
  p.q_start = a.q_start;
  p.q = (const uint16_t*)a.q; p.k = (const uint16_t*)a.k; p.v = (const uint16_t*)a.v;
  p.wq = (const uint16_t*)a.wq; p.wk = (const uint16_t*)a.wk;
  p.eps = a.eps;
  p.q_out = (uint16_t*)a.q_out;
  p.k_pages = (uint8_t*)a.k_pages; p.v_pages = (uint8_t*)a.v_pages;
  p.k_scale = a.k_scale; p.v_scale = a.v_scale;
  p.page_table = a.page_table;
  p.seq_pos = a.seq_pos;
  p.status = a.status;
  if (a.rope) {
    p.cos = a.rope->cos; p.sin = a.rope->sin;
    p.positions = a.rope->positions; p.pair_axis = a.rope->pair_axis;
    p.n_positions = a.rope->n_positions; p.n_axes = a.rope->n_axes; p.rot = a.rope->rotary_dim;
  }
  const long long q_rows = a.q ? (long long)g.n_layers * a.n_tokens : 0;
  if (!a.q_start) {
    const long long warps = (long long)g.n_layers * g.batch * g.h_kv * 2 + q_rows;
    const long long grid = (warps + 7) / 8;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (g.head_dim == 128) paged_append_token_kernel<128><<<(unsigned)grid, 256, 0, stream>>>(p);
    else paged_append_token_kernel<256><<<(unsigned)grid, 256, 0, stream>>>(p);
  } else if (a.n_tokens > 0) {
    // pages that the call touches: n tokens touch at most n pages, and at most n / page_size + 2 (an open first and last page)
    const long long most = (long long)a.n_tokens / g.page_size + 2LL * g.batch;
    p.kv_blocks = (int)(most < a.n_tokens ? most : a.n_tokens);
    const int threads = g.page_size * g.head_dim == 128 * 256 ? 512 : 256;
    const long long grid = (long long)p.kv_blocks * g.h_kv * 2 * g.n_layers + (q_rows + threads / 32 - 1) / (threads / 32);
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    auto launch = [&](auto kernel) { kernel<<<(unsigned)grid, threads, 0, stream>>>(p); };
    if (g.head_dim == 128) {
      switch (g.page_size) {
        case 16: launch(paged_append_prompt_kernel<128, 1, 256>); break;
        case 32: launch(paged_append_prompt_kernel<128, 2, 256>); break;
        case 64: launch(paged_append_prompt_kernel<128, 4, 256>); break;
        default: launch(paged_append_prompt_kernel<128, 8, 256>); break;
      }
    } else {
      switch (g.page_size) {
        case 16: launch(paged_append_prompt_kernel<256, 2, 256>); break;
        case 32: launch(paged_append_prompt_kernel<256, 4, 256>); break;
        case 64: launch(paged_append_prompt_kernel<256, 8, 256>); break;
        default: launch(paged_append_prompt_kernel<256, 8, 512>); break;
      }
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (a.advance_pos) {
    paged_advance_kernel<<<(g.batch + 127) / 128, 128, 0, stream>>>(g, a.q_start, a.seq_pos);
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace b200attn
