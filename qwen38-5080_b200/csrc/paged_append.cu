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
// Bound: HBM bytes (query in and out, key and value in, bytes out), and for single tokens the launch.  A 32768-token prompt of 40 / 8
// heads: 164 us, of which queries 108 (6.2 TB/s) and keys and values 55 (3.7 TB/s: issue slots, and a barrier per page and head); one
// token of 64 layers x 16 sequences: 7.5 us (3.6 TB/s).
#include "paged.cuh"
#include "streamk.cuh"

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
  int q_run;                              // groups of query heads that a warp takes in turn
  uint32_t q_units;       // warps' shares of the queries
  int kv_blocks, heads;   // pages that the call touches, at most; kv heads that a block takes in turn
};

// Smallest power of two s with amax / s <= 448 = 1.75 * 2^8, at least 2^-126; amax is finite and >= 0.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // biased exponent of s
  return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}

constexpr float kFltMax = 3.402823466e38f;
// Largest of the warp's values; none is negative, so their bits compare as integers.
__device__ __forceinline__ float warp_max(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); }
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= kFltMax ? a : 0.f;   // NaN and infinities do not take part in the maximum
}

// A lane's share of a head row: four dims at `a` and four at `b`.  In the rotated part b = a + R / 2: a lane holds both halves of
// its four pairs, so that the rotation needs no other lane (16 contiguous bytes per lane instead made 8 shuffles and twice the
// cosines and sines: 170 instructions per 8 values, and the kernels were bound by issue).  Beyond it, 8 dims in a row.
template <int D>
struct Share {
  static constexpr int TPR = D / 8;   // lanes per head row
  int a, b;
  bool on;                            // rotated
  __device__ __forceinline__ Share(int lane, int rot) {
    const int l = lane % TPR;
    on = 8 * l < rot;
    a = on ? 4 * l : 8 * l;
    b = a + (on ? rot >> 1 : 4);
  }
};
struct Raw { uint2 a, b; };
// Read once: not worth a line of L1.
__device__ __forceinline__ uint2 ldg_once(const uint16_t* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
template <int D>
__device__ __forceinline__ Raw load_row(const uint16_t* row, const Share<D>& sh) { return Raw{ldg_once(row + sh.a), ldg_once(row + sh.b)}; }
__device__ __forceinline__ void unpack(const Raw& r, float (&x)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint2 pack4(const float* x) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]), q = __floats2bfloat162_rn(x[2], x[3]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
}
// 1 / s, of a power of two by its exponent (scales that the append made are)
__device__ __forceinline__ float reciprocal(float s) {
  const uint32_t bits = __float_as_uint(s), e = bits >> 23;
  return (bits & 0x7FFFFFu) == 0 && e >= 1 && e < 254 ? __uint_as_float((254u - e) << 23) : __fdiv_rn(1.f, s);
}
// 4 floats -> 4 e4m3 bytes: nearest even, saturating at 448; NaN -> 0x7F
__device__ __forceinline__ uint32_t quant4(const float* x, float inv) {
  uint32_t bytes;
  float x0, x1, x2, x3;
  split2(mul2(pair2(x[0], x[1]), pair2(inv, inv)), x0, x1);
  split2(mul2(pair2(x[2], x[3]), pair2(inv, inv)), x2, x3);
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}" : "=r"(bytes) : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
  return bytes;
}
// 16 e4m3 bytes re-expressed in a larger power-of-two scale: value * ratio, ratio = old / new < 1
__device__ __forceinline__ uint4 rescale16(const uint4& raw, float ratio) {
  float f[16];
  e4m3x16_to_float(raw, f);
  return make_uint4(quant4(f, ratio), quant4(f + 4, ratio), quant4(f + 8, ratio), quant4(f + 12, ratio));
}

// The cosines and sines of a lane's four pairs for one token (lanes beyond the rotated dims load those of pair 0 and do not use
// them, so that no load stands behind a branch).
struct Rotation {
  float4 c, s;

  __device__ __forceinline__ int clamped(const AppendParams& p, int pos, bool bad, bool on) const {
    bad |= pos < 0 || pos >= p.n_positions;
    if (bad && on) atomicOr(p.status, B200ATTN_STATUS_BAD_POSITION);
    return min(max(pos, 0), p.n_positions - 1);
  }
  template <int D>
  __device__ __forceinline__ void load(const AppendParams& p, const Share<D>& sh, int token, int slot) {
    if (p.rot == 0) return;
    const int half = p.rot >> 1, j0 = sh.on ? sh.a : 0;
    if (p.pair_axis == nullptr) {
      const int pos = clamped(p, p.positions ? ld(p.positions + token) : slot, false, sh.on);
      B200ATTN_CHECK(p.status, pos >= 0 && pos < p.n_positions && j0 + 4 <= half);
      c = ld(reinterpret_cast<const float4*>(p.cos + (long long)pos * half + j0));
      s = ld(reinterpret_cast<const float4*>(p.sin + (long long)pos * half + j0));
    } else {
      const int4 ax = ld(reinterpret_cast<const int4*>(p.pair_axis + j0));
      int at[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) at[a] = !p.positions ? slot : a < p.n_axes ? ld(p.positions + (long long)a * p.n_tokens + token) : 0;
      auto pick = [&](int a) { return (long long)clamped(p, a == 1 ? at[1] : a == 2 ? at[2] : a == 3 ? at[3] : at[0], a < 0 || a >= p.n_axes, sh.on) * half + j0; };
      const long long i0 = pick(ax.x), i1 = pick(ax.y) + 1, i2 = pick(ax.z) + 2, i3 = pick(ax.w) + 3;
      B200ATTN_CHECK(p.status, i0 >= 0 && i1 >= 0 && i2 >= 0 && i3 >= 0 && max(max(i0, i1), max(i2, i3)) < (long long)p.n_positions * half);
      c = make_float4(ld(p.cos + i0), ld(p.cos + i1), ld(p.cos + i2), ld(p.cos + i3));
      s = make_float4(ld(p.sin + i0), ld(p.sin + i1), ld(p.sin + i2), ld(p.sin + i3));
    }
  }
  __device__ __forceinline__ void turn(float (&x)[8]) const {
    const unsigned long long cc[2] = {pair2(c.x, c.y), pair2(c.z, c.w)}, ss[2] = {pair2(s.x, s.y), pair2(s.z, s.w)};
    const unsigned long long nn[2] = {pair2(-s.x, -s.y), pair2(-s.z, -s.w)};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const unsigned long long u = pair2(x[2 * e], x[2 * e + 1]), v = pair2(x[4 + 2 * e], x[5 + 2 * e]);
      split2(fma2(u, cc[e], mul2(v, nn[e])), x[2 * e], x[2 * e + 1]);
      split2(fma2(v, cc[e], mul2(u, ss[e])), x[4 + 2 * e], x[5 + 2 * e]);
    }
  }
};

// RMS norm over the head's lanes; every lane of the warp calls it.
template <int D>
__device__ __forceinline__ void rms_norm(float (&x)[8], const float (&w1)[8], float eps) {
  unsigned long long y[4], sum = 0ull;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = pair2(x[2 * e], x[2 * e + 1]);
    sum = fma2(y[e], y[e], sum);
  }
  float ss, odd;
  split2(sum, ss, odd);
  ss += odd;
#pragma unroll
  for (int off = D / 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  const float inv = __frsqrt_rn(ss * (1.f / D) + eps);
  const unsigned long long inv2 = pair2(inv, inv);
#pragma unroll
  for (int e = 0; e < 4; ++e) split2(mul2(mul2(y[e], inv2), pair2(w1[2 * e], w1[2 * e + 1])), x[2 * e], x[2 * e + 1]);
}
template <int D>
__device__ __forceinline__ void load_norm(const uint16_t* w, int layer, const Share<D>& sh, float (&w1)[8]) {
  const uint16_t* row = w + (long long)layer * D;
  const Raw r{ld(reinterpret_cast<const uint2*>(row + sh.a)), ld(reinterpret_cast<const uint2*>(row + sh.b))};
  unpack(r, w1);
#pragma unroll
  for (int e = 0; e < 8; ++e) w1[e] += 1.f;
}

// Sequence that owns packed token t (largest b with q_start[b] <= t; empty sequences share their start).
__device__ __forceinline__ int sequence_of(const int* q_start, int batch, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ld(q_start + mid) <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int page_of(const AppendParams& p, int b, int page_index) {
  const int id = p.page_table[(long long)b * p.g.max_pages + page_index];
  return id >= 0 && id < p.g.n_pages ? id : -1;
}

// Query rows: a warp takes kQLoads loads' worth of a token's heads at a time, all in flight together, and rotates them with one set
// of cosines and sines.  (One warp per token, head after head, waited for every load: 445 us for a 32768-token prompt of 40 / 8
// heads against 160 us for its keys and values alone.)  Where there are many tokens it goes on with the token's next heads, whose
// rows are on their way meanwhile: finding the token's sequence, position and angles is half of the instructions otherwise.
constexpr int kQLoads = 4;
template <int D>
__host__ __device__ constexpr int q_heads() { return kQLoads * 32 / (D / 8); }   // heads of a group: 8 or 4
template <int D, bool RUN>   // RUN: several groups in turn
__device__ __forceinline__ void rotate_queries(const AppendParams& p, uint32_t unit) {
  constexpr int TPR = D / 8, RPW = 32 / TPR;   // lanes per head row, rows per load
  const int lane = threadIdx.x & 31;
  const int groups = (p.g.h_q + q_heads<D>() - 1) / q_heads<D>();
  const int run = RUN ? p.q_run : 1;
  const uint32_t chunks = (uint32_t)(groups + run - 1) / run;
  const uint32_t r = unit / chunks;            // (layer, token)
  const int g_first = (int)(unit - r * chunks) * run, g_end = min(groups, g_first + run);
  const int layer = (int)(r / (uint32_t)p.n_tokens), token = (int)(r - (uint32_t)layer * p.n_tokens);
  B200ATTN_CHECK(p.status, layer < p.g.n_layers && token < p.n_tokens && g_first < groups);
  const Share<D> sh(lane, p.rot);
  B200ATTN_CHECK(p.status, sh.a >= 0 && sh.b + 4 <= D && (!sh.on || sh.b + 4 <= p.rot));
  const long long row0 = (long long)r * p.g.h_q + lane / TPR;
  Raw raw[kQLoads];
  auto load = [&](int group) {
#pragma unroll
    for (int i = 0; i < kQLoads; ++i) {
      const int h = group * q_heads<D>() + i * RPW;
      if (h + lane / TPR < p.g.h_q) raw[i] = load_row<D>(p.q + (row0 + h) * D, sh);
    }
  };
  load(g_first);
  int b = token, slot;
  if (p.q_start) {
    if (token >= ld(p.q_start + p.g.batch) || token < ld(p.q_start)) return;   // a row that belongs to nobody
    b = sequence_of(p.q_start, p.g.batch, token);
    slot = (int)min((long long)ld(p.seq_pos + b) + token - ld(p.q_start + b), 0x7fffffffLL);
  } else {
    slot = ld(p.seq_pos + b);
  }
  Rotation rot;
  rot.load<D>(p, sh, token, slot);
  float w1[8];
  if (p.wq) load_norm<D>(p.wq, layer, sh, w1);
#pragma unroll 1
  for (int group = g_first; group < (RUN ? g_end : g_first + 1); ++group) {
    Raw now[kQLoads];
#pragma unroll
    for (int i = 0; i < kQLoads; ++i) now[i] = raw[i];
    if (RUN && group + 1 < g_end) load(group + 1);
#pragma unroll
    for (int i = 0; i < kQLoads; ++i) {
      float x[8];
      unpack(now[i], x);
      if (p.wq) rms_norm<D>(x, w1, p.eps);
      if (sh.on) rot.turn(x);
      const int h = group * q_heads<D>() + i * RPW;
      if (h + lane / TPR < p.g.h_q) {
        uint16_t* dst = p.q_out + (row0 + h) * D;
        *reinterpret_cast<uint2*>(dst + sh.a) = pack4(x);
        *reinterpret_cast<uint2*>(dst + sh.b) = pack4(x + 4);
      }
    }
  }
}

// One token per sequence.  D / 8 lanes hold a key or value row: half a warp the key and half the value of a head (heads of
// 128), or a warp one of them (256).  The same lanes re-express the page's earlier rows when the scale grows.  The warps behind
// those rotate the queries.
template <int D>
__global__ void __launch_bounds__(128)
paged_append_token_kernel(const AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int TPR = D / 8, RPW = 32 / TPR;
  const PagedGeometry& g = p.g;
  const int lane = threadIdx.x & 31, lr = lane % TPR;
  const uint32_t warp = blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint32_t rows = (uint32_t)g.n_layers * g.batch * g.h_kv * 2, kv_warps = (rows + RPW - 1) / RPW;   // rows is even
  if (warp >= kv_warps) {
    if (warp - kv_warps < p.q_units) rotate_queries<D, false>(p, warp - kv_warps);
    return;
  }
  const uint32_t r2 = warp * RPW + lane / TPR;       // (layer, sequence, head, key or value)
  const int which = (int)(r2 & 1);                   // 0 key, 1 value
  const uint32_t row = r2 >> 1;
  const int h = (int)(row % g.h_kv);
  const uint32_t lb = row / g.h_kv;
  const int b = (int)(lb % g.batch), layer = (int)(lb / g.batch);
  const Share<D> sh(lane, p.rot);
  const Raw raw = load_row<D>((which ? p.v : p.k) + (long long)row * D, sh);
  const int pos = ld(p.seq_pos + b);
  const bool fits = pos >= 0 && pos < (long long)g.max_pages * g.page_size;
  const int page = fits ? page_of(p, b, pos / g.page_size) : -1, fill = fits ? pos % g.page_size : 0;
  // a sequence without a token and without a page (-1) is idle: nothing to store, nothing to report
  if (page < 0 && lr == 0 && (pos != 0 || ld(p.page_table + (long long)b * g.max_pages) != -1))
    atomicOr(p.status, fits ? B200ATTN_STATUS_BAD_PAGE : B200ATTN_STATUS_POS_AT_CAPACITY);
  float* sp = (which ? p.v_scale : p.k_scale) + ((long long)layer * g.n_pages + page) * g.h_kv + h;
  const float old = page >= 0 && fill > 0 ? *sp : 0.f;
  float x[8];
  unpack(raw, x);
  if (RPW == 2 || !which) {                          // uniform over the warp: it holds a key and a value, or one of them
    if (p.wk) {
      float w1[8], k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = x[e];
      load_norm<D>(p.wk, layer, sh, w1);
      rms_norm<D>(k, w1, p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = which ? x[e] : k[e];
    }
    Rotation rot;
    rot.load<D>(p, sh, b, fits ? pos : 0);
    if (!which && sh.on) rot.turn(x);
  }
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(x[e]));
#pragma unroll
  for (int off = TPR / 2; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if (page < 0) return;
  float s = pow2_scale(amax);
  uint8_t* base = (which ? p.v_pages : p.k_pages) + (long long)layer * (which ? g.v_layer_stride : g.k_layer_stride) +
                  ((long long)page * g.h_kv + h) * g.page_size * D;
  if (fill > 0) {
    if (s > old) {
      const float ratio = old / s;
      uint4* rows16 = reinterpret_cast<uint4*>(base);
      const int n = fill * (D / 16);
#pragma unroll 4
      for (int i = lr; i < n; i += TPR) rows16[i] = rescale16(rows16[i], ratio);
    } else {
      s = old;
    }
  }
  if (lr == 0) *sp = s;
  const float inv = __fdiv_rn(1.f, s);
  B200ATTN_CHECK(p.status, r2 < rows && rows_exist(g, ((long long)page * g.h_kv + h) * g.page_size + fill, 1, layer) && fill < g.page_size);
  uint8_t* dst = base + (long long)fill * D;
  *reinterpret_cast<uint32_t*>(dst + sh.a) = quant4(x, inv);
  *reinterpret_cast<uint32_t*>(dst + sh.b) = quant4(x + 4, inv);
}

// Prompts.  A thread block holds the new tokens of one page for `heads` kv heads in turn, of keys or of values: it rotates
// them, finds the page's scale, writes them; the next head's rows are on their way meanwhile.  THREADS x NP rows' shares cover a
// page.
template <int D, int NP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
paged_append_prompt_kernel(const AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int TPR = D / 8, RPP = THREADS / TPR;
  const PagedGeometry& g = p.g;
  const int tid = threadIdx.x, lane = tid & 31;
  const int groups = (g.h_kv + p.heads - 1) / p.heads;
  const int which = (int)(blockIdx.x & 1);
  uint32_t u = blockIdx.x >> 1;
  const int h_first = (int)(u % groups) * p.heads, h_end = min(h_first + p.heads, g.h_kv);
  u /= groups;
  const int chunk = (int)(u % p.kv_blocks), layer = (int)(u / p.kv_blocks);

  // the sequence and page that chunk number `chunk` of the call is: a scan over the sequences' touched pages
  __shared__ int s_at[5];                                // sequence, page of it, first packed token, tokens, tokens before
  __shared__ float s_max[2][THREADS / 32];
  if (tid < 32) {
    int before = 0;
    if (tid == 0) s_at[0] = -1;
    __syncwarp();
    for (int b0 = 0; b0 < g.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0, first = 0, q0 = 0, nt = 0, pos = 0;
      if (b < g.batch) {
        q0 = p.q_start[b];
        const int end = p.q_start[b + 1];
        nt = end - q0;
        pos = p.seq_pos[b];
        const bool fits = range_fits(q0, end, p.n_tokens, p.status, blockIdx.x == 0);
        if (fits && nt > 0 && pos < 0 && blockIdx.x == 0) atomicOr(p.status, B200ATTN_STATUS_BAD_POSITION);
        if (fits && nt > 0 && pos >= 0) {
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
      if (n > 0 && chunk >= start && chunk < start + n) { s_at[0] = b; s_at[1] = first + chunk - start; s_at[2] = q0; s_at[3] = nt; s_at[4] = pos; }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > chunk && blockIdx.x != 0) break;          // the first block has looked at every sequence
    }
  }
  __syncthreads();
  const int b = s_at[0];
  if (b < 0) return;                                     // the grid is an upper bound
  const int page_index = s_at[1], q0 = s_at[2], nt = s_at[3], pos = s_at[4];
  if (page_index >= g.max_pages) {                       // before anything is computed from it: slots behind the table can pass 31 bits
    if (tid == 0) atomicOr(p.status, B200ATTN_STATUS_POS_AT_CAPACITY);
    return;
  }
  const int slot0 = page_index * g.page_size;
  const int lo = max(pos - slot0, 0);                                                   // rows [lo, hi) are new
  const int hi = (int)min((long long)g.page_size, (long long)pos + nt - slot0);
  const Share<D> sh(lane, p.rot);
  // the thread's first row of the next head, and whether its rows are new (addresses by addition: computed anew for every row and head
  // they were a third of the kernel's instructions)
  const uint16_t* src = (which ? p.v : p.k) + (((long long)layer * p.n_tokens + q0 + slot0 - pos + tid / TPR) * g.h_kv + h_first) * D;
  const int row_step = RPP * g.h_kv * D;
  bool is_new[NP];
  Raw raw[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = i * RPP + tid / TPR;
    is_new[i] = row >= lo && row < hi;
    raw[i] = Raw{make_uint2(0, 0), make_uint2(0, 0)};     // rows that are not new stay zero
    B200ATTN_CHECK(p.status, !is_new[i] || (slot0 + row >= pos && slot0 + row < pos + nt && q0 + slot0 + row - pos < p.n_tokens));
  }
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (is_new[i]) raw[i] = load_row<D>(src + i * row_step, sh);
    src += D;
  };
  load();
  const int page = page_of(p, b, page_index);
  if (page < 0) {
    if (tid == 0) atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE);
    return;
  }
  Rotation rot[NP];                                      // of this thread's rows, for all heads
  if (!which)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = min(max(i * RPP + tid / TPR, lo), hi - 1);
      rot[i].load<D>(p, sh, q0 + slot0 + row - pos, slot0 + row);
    }
  float* scales = (which ? p.v_scale : p.k_scale) + ((long long)layer * g.n_pages + page) * g.h_kv;
  uint8_t* base = (which ? p.v_pages : p.k_pages) + (long long)layer * (which ? g.v_layer_stride : g.k_layer_stride) +
                   ((long long)page * g.h_kv + h_first) * g.page_size * D;   // the page of the head
  B200ATTN_CHECK(p.status, lo >= 0 && lo < hi && hi <= g.page_size && RPP * NP >= g.page_size &&
                               rows_exist(g, ((long long)page * g.h_kv + h_first) * g.page_size, (h_end - h_first) * g.page_size, layer));
#pragma unroll 1
  for (int h = h_first; h < h_end; ++h, base += g.page_size * D) {
    float x[NP][8];
#pragma unroll
    for (int i = 0; i < NP; ++i) unpack(raw[i], x[i]);
    const float old = lo > 0 ? scales[h] : 0.f;
    if (h + 1 < h_end) load();
    if (!which && p.wk) {
      float w1[8];
      load_norm<D>(p.wk, layer, sh, w1);
#pragma unroll
      for (int i = 0; i < NP; ++i) rms_norm<D>(x[i], w1, p.eps);
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (!which && sh.on) rot[i].turn(x[i]);
#pragma unroll
      for (int e = 0; e < 8; e += 2) amax = max3(amax, fabsf(x[i][e]), fabsf(x[i][e + 1]));   // NaN is passed over
    }
    amax = warp_max(amax);
    if (amax > kFltMax) {                                 // infinities among them: once more without
      amax = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(x[i][e]));
      amax = warp_max(amax);
    }
    if (lane == 0) s_max[h & 1][tid >> 5] = amax;
    __syncthreads();                                      // maxima are in; every thread has read the old scale
    amax = warp_max(lane < THREADS / 32 ? s_max[h & 1][lane] : 0.f);
    float s = pow2_scale(amax);
    if (lo > 0) {
      if (s > old) {
        const float ratio = old / s;
        uint4* rows16 = reinterpret_cast<uint4*>(base);
        for (int i = tid; i < lo * (D / 16); i += THREADS) rows16[i] = rescale16(rows16[i], ratio);
      } else {
        s = old;
      }
    }
    if (tid == 0) scales[h] = s;
    const float inv = reciprocal(s);
    uint8_t* rows = base + tid / TPR * D;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (is_new[i]) {
        uint8_t* dst = rows + i * RPP * D;
        *reinterpret_cast<uint32_t*>(dst + sh.a) = quant4(x[i], inv);
        *reinterpret_cast<uint32_t*>(dst + sh.b) = quant4(x[i] + 4, inv);
      }
    }
  }
}

// The queries of prompts: a kernel of their own, with more warps on an SM than the one above has.  (Blocks of 256 threads, three to an SM:
// 46.5 us for 7,500 tokens of 24 heads of 256 with norms, against 44.4.)
constexpr int kQThreads = 128;
template <int D>
__global__ void __launch_bounds__(kQThreads, 6) paged_rotate_queries_kernel(const AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t unit = blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5);
  if (unit < p.q_units) rotate_queries<D, true>(p, unit);
}

// A warp per sequence: its position moves on if every new token has found a page.
__global__ void paged_advance_kernel(PagedGeometry g, int n_tokens, const int* q_start, const int* page_table, int* seq_pos) {
  pdl_wait();
  const int b = (int)(blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (b >= g.batch) return;
  const int q0 = q_start ? q_start[b] : b, end = q_start ? q_start[b + 1] : b + 1, pos = seq_pos[b];
  if (q0 < 0 || end <= q0 || end > n_tokens || pos < 0 || (long long)pos + (end - q0) > (long long)g.max_pages * g.page_size) return;
  const int last = (pos + (end - q0) - 1) / g.page_size;
  bool there = true;
  for (int i = pos / g.page_size + lane; i <= last; i += 32) {
    const int id = page_table[(long long)b * g.max_pages + i];
    there &= id >= 0 && id < g.n_pages;
  }
  if (__all_sync(0xffffffffu, there) && lane == 0) seq_pos[b] = pos + (end - q0);
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
  const int q_heads_ = g.head_dim == 128 ? q_heads<128>() : q_heads<256>();
  // groups of heads that a warp takes in turn: as many as leave an SM 64 warps of queries
  const int groups = (g.h_q + q_heads_ - 1) / q_heads_;
  const long long run = (long long)g.n_layers * a.n_tokens * groups / (64LL * device_sms());
  const int chunks = run <= 1 ? groups : run >= groups ? 1 : (groups + (int)run - 1) / (int)run;
  p.q_run = a.q_start ? (groups + chunks - 1) / chunks : 1;
  const long long q_warps = a.q ? (long long)g.n_layers * a.n_tokens * ((groups + p.q_run - 1) / p.q_run) : 0;
  const long long kv_rows = (long long)g.n_layers * g.batch * g.h_kv * 2;
  if (q_warps > 0x7fffffffLL || kv_rows > 0x7fffffffLL) return cudaErrorInvalidConfiguration;   // indices are 32-bit
  p.q_units = (uint32_t)q_warps;
  cudaError_t e = cudaSuccess;
  if (!a.q_start) {
    const long long rpw = g.head_dim == 128 ? 2 : 1, grid = ((kv_rows + rpw - 1) / rpw + q_warps + 3) / 4;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    e = g.head_dim == 128 ? launch_pdl(paged_append_token_kernel<128>, (int)grid, 128, 0, stream, p)
                          : launch_pdl(paged_append_token_kernel<256>, (int)grid, 128, 0, stream, p);
  } else if (a.n_tokens > 0) {
    // pages that the call touches: n tokens touch at most n pages, and at most n / page_size + 2 (an open first and last page)
    const long long most = (long long)a.n_tokens / g.page_size + 2LL * g.batch;
    p.kv_blocks = (int)(most < a.n_tokens ? most : a.n_tokens);
    // two loads of 16 bytes per thread and page (four for the largest pages); of its heads a block takes as many in turn as leave every SM a few blocks
    const int threads = g.page_size * g.head_dim / 16 < 1024 ? g.page_size * g.head_dim / 16 : 1024;
    const long long pages = (long long)p.kv_blocks * 2 * g.n_layers, blocks = 2LL * device_sms() * (1024 / threads);
    long long heads = pages * g.h_kv / blocks;
    p.heads = (int)(heads < 1 ? 1 : heads > g.h_kv ? g.h_kv : heads);
    const long long grid = pages * ((g.h_kv + p.heads - 1) / p.heads), q_grid = (q_warps + kQThreads / 32 - 1) / (kQThreads / 32);
    if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (q_grid) {
      e = g.head_dim == 128 ? launch_pdl(paged_rotate_queries_kernel<128>, (int)q_grid, kQThreads, 0, stream, p)
                            : launch_pdl(paged_rotate_queries_kernel<256>, (int)q_grid, kQThreads, 0, stream, p);
      if (e != cudaSuccess) return e;
    }
    auto launch = [&](auto kernel) { e = launch_pdl(kernel, (int)grid, threads, 0, stream, p); };
    if (g.head_dim == 128) {
      switch (g.page_size) {
        case 16: launch(paged_append_prompt_kernel<128, 2, 128>); break;
        case 32: launch(paged_append_prompt_kernel<128, 2, 256>); break;
        case 64: launch(paged_append_prompt_kernel<128, 2, 512>); break;
        default: launch(paged_append_prompt_kernel<128, 2, 1024>); break;
      }
    } else {
      switch (g.page_size) {
        case 16: launch(paged_append_prompt_kernel<256, 2, 256>); break;
        case 32: launch(paged_append_prompt_kernel<256, 2, 512>); break;
        case 64: launch(paged_append_prompt_kernel<256, 2, 1024>); break;
        default: launch(paged_append_prompt_kernel<256, 4, 1024>); break;
      }
    }
  }
  if (e == cudaSuccess && a.advance_pos)
    e = launch_pdl(paged_advance_kernel, (g.batch + 3) / 4, 128, 0, stream, g, a.n_tokens, a.q_start, a.page_table, a.seq_pos);
  return e;
}

}  // namespace b200attn
