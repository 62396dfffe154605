// Attention of one query token per sequence over the paged FP8 cache: one scale per (page, kv head).
//
//   s_t = (q . k_t) * k_scale[page(t)] * softmax_scale * log2(e),   out = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m)
//
// Bound: HBM.  Every K and V byte of the attended tokens is read once and serves all G <= 8 query heads of its kv head.
//
// A thread block of four warps takes a piece of one (layer, sequence, kv head) pair; a warp takes 16 tokens at a time,
// straight from global memory into registers in the layout that the tensor core wants, so there is nothing to fill, no
// barrier in the loop and no wait at its start: what counts for a single layer of one user is latency, and for long
// caches sixteen warps per SM keep about 50 KB of loads in flight.
//   * S^T[16 tokens x 8 heads] = K q^T: mma.m16n8k16 with K widened to f16 (exact).  The order of the head dims is free as
//     long as K and q agree: a lane's 16-byte load is 16 of "its" dims, and a warp's load is 64 bytes of 8 rows each.
//   * O^T[D x 8 heads] += V^T P^T: a lane loads the same 16 dims of four tokens (a warp: four whole rows) and pairs the
//     tokens' bytes; P^T comes from a movmatrix transpose.
//   * K registers are reloaded for the warp's next tokens as soon as the scores are done, V registers as soon as the
//     product is: both loads stay in flight under the other half of the work.
// Precision: q is scaled by a power of two per head and held in f16, exact for every bf16 within 2^14 of the head's
// largest value.  p * 2^15 is held in f16 (11 bits, down to 2^-39 of the largest): a rounding of 2^-12 per token against
// the output's 2^-9.  The page's V scale goes into p relative to the largest V scale so far (r): p * v_scale / r <= p.
// Sums and accumulators are fp32.
//
// Long sequences are cut into pieces over several thread blocks.  Each leaves (m, l, O) in the workspace and takes a
// ticket; the last one joins the pieces in order, so the result does not depend on who is last, and sets the counter
// back to zero.  Nobody waits for anybody.
#include "paged.cuh"

namespace b200attn {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16 * kWarps;        // tokens the block takes per round
constexpr int kStage = 256;               // pages whose number and scales are in shared memory at a time
constexpr float kPBits = 15.f;            // p is held times 2^15

struct DecodeParams {
  PagedGeometry g;
  const uint16_t* q;
  const uint8_t *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int *page_table, *seq_len;
  int seq_len_offset;
  float score_scale;                      // softmax_scale * log2(e)
  int num_splits;
  float* part;                            // [pairs][num_splits][G * D + 16]: O, m[8], l[8]
  int* counters;                          // [pairs]
  uint16_t* out;
  int* status;
};

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) { return e4m3x2_to_f16x2((uint16_t)(w & 0xFFFFu)); }
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) { return e4m3x2_to_f16x2((uint16_t)(w >> 16)); }
__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int D>
__global__ void __launch_bounds__(kThreads, D == 128 ? 4 : 2)
paged_decode_kernel(const DecodeParams p) {
  constexpr int KS = D / 16;              // k-steps of the score product, dim tiles of the output product
  constexpr int KL = D / 64;              // 16-byte loads per K row and lane
  constexpr int DH = D / 128;             // 128-byte halves of a V row
  const PagedGeometry& g = p.g;
  const int G = g.group;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
  const long long pair = blockIdx.x / p.num_splits;
  const int split = (int)(blockIdx.x % p.num_splits);
  const int h = (int)(pair % g.h_kv);
  const long long lb = pair / g.h_kv;
  const int b = (int)(lb % g.batch), layer = (int)(lb / g.batch);

  __shared__ int s_page[kStage];
  __shared__ float2 s_scale[kStage];
  __shared__ float s_ml[kWarps][2][8];
  __shared__ int s_last;
  extern __shared__ float s_acc[];        // [kWarps][G][D]

  const int len = paged_len(g, p.seq_len[b] + p.seq_len_offset, p.status, tid == 0 && split == 0 && h == 0 && layer == 0);
  // pieces: as many as the grid has room for, each a whole number of rounds
  const int rounds = (len + kUnit - 1) / kUnit;
  const int per = (rounds + p.num_splits - 1) / p.num_splits;
  const int pieces = per > 0 ? (rounds + per - 1) / per : 0;
  if (split >= pieces) {
    if (pieces == 0 && split == 0)        // no tokens: zeros
      for (int i = tid; i < G * D / 2; i += kThreads)
        reinterpret_cast<uint32_t*>(p.out + (lb * g.h_q + h * G) * D)[i] = 0u;
    return;
  }
  const int t_begin = split * per * kUnit, t_end = min(len, t_begin + per * kUnit);

  // ---- query fragments: lane holds head gq, dims 16 * (4 ch + tq) + 4 w + {0, 1 | 2, 3} ----
  uint32_t qf[KS][2];
  float sc0, sc1;                         // score multipliers of heads 2 tq, 2 tq + 1
  {
    float x[KL][16];
    float amax = 0.f;
    const uint16_t* qp = p.q + (lb * g.h_q + h * G + gq) * D + tq * 16;
#pragma unroll
    for (int ch = 0; ch < KL; ++ch)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (gq < G) raw = *reinterpret_cast<const uint4*>(qp + ch * 64 + i * 8);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[ch][8 * i + 2 * e] = bf16_bits_to_float(w[e] & 0xFFFFu);
          x[ch][8 * i + 2 * e + 1] = bf16_bits_to_float(w[e] >> 16);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[ch][8 * i + e]));
      }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    int ex = (int)((__float_as_uint(amax) >> 23) & 0xFF);
    ex = ex < 1 ? 1 : (ex > 253 ? 253 : ex);
    const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
    for (int ch = 0; ch < KL; ++ch)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const __half2 b0 = __floats2half2_rn(x[ch][4 * w] * down, x[ch][4 * w + 1] * down);
        const __half2 b1 = __floats2half2_rn(x[ch][4 * w + 2] * down, x[ch][4 * w + 3] * down);
        qf[ch * 4 + w][0] = *reinterpret_cast<const uint32_t*>(&b0);
        qf[ch * 4 + w][1] = *reinterpret_cast<const uint32_t*>(&b1);
      }
    const float mult = up * p.score_scale;
    sc0 = __shfl_sync(0xffffffffu, mult, 8 * tq);
    sc1 = __shfl_sync(0xffffffffu, mult, 8 * tq + 4);
  }

  const uint8_t* kbase = p.k_pages + (long long)layer * g.k_layer_stride;
  const uint8_t* vbase = p.v_pages + (long long)layer * g.v_layer_stride;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, r = 0.f, inv_r = 0.f;
  float o[KS][4];
#pragma unroll
  for (int j = 0; j < KS; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f; }

  const int block_tokens = kStage * g.page_size;
  for (int t_stage = t_begin / g.page_size * g.page_size; t_stage < t_end; t_stage += block_tokens) {
    // ---- the pages of this stretch: their numbers and scales ----
    if (t_stage > t_begin) __syncthreads();
    const int first = t_stage / g.page_size, stage_end = min(t_end, t_stage + block_tokens);
    for (int i = tid; i < (stage_end - t_stage + g.page_size - 1) / g.page_size; i += kThreads) {
      int id = p.page_table[(long long)b * g.max_pages + first + i];
      float2 sc = make_float2(0.f, 0.f);
      if (id < 0 || id >= g.n_pages) {
        atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE);
        id = -1;
      } else {
        const long long si = ((long long)layer * g.n_pages + id) * g.h_kv + h;
        sc = make_float2(p.k_scale[si], p.v_scale[si]);
      }
      s_page[i] = id;
      s_scale[i] = sc;
    }
    __syncthreads();

    uint4 kr[KL][2], vr[DH][4];
    int tok = max(t_begin, t_stage) + warp * 16;
    // offset of a 16-token step's rows, or -1: no tokens there, or a page that does not exist
    auto rows_of = [&](int t) -> long long {
      if (t >= stage_end) return -1;
      const int id = s_page[t / g.page_size - first];
      return id < 0 ? -1 : (((long long)id * g.h_kv + h) * g.page_size + t % g.page_size) * D;
    };
    auto load_k = [&](long long off) {
      if (off < 0) return;
      const uint8_t* src = kbase + off + gq * D + tq * 16;
#pragma unroll
      for (int ch = 0; ch < KL; ++ch) {
        kr[ch][0] = ldg_stream(src + ch * 64);
        kr[ch][1] = ldg_stream(src + ch * 64 + 8 * D);
      }
    };
    auto load_v = [&](long long off) {
      if (off < 0) return;
      const uint8_t* src = vbase + off + 2 * tq * D + gq * 16;
#pragma unroll
      for (int hf = 0; hf < DH; ++hf) {
        vr[hf][0] = ldg_stream(src + hf * 128);
        vr[hf][1] = ldg_stream(src + hf * 128 + D);
        vr[hf][2] = ldg_stream(src + hf * 128 + 8 * D);
        vr[hf][3] = ldg_stream(src + hf * 128 + 9 * D);
      }
    };
    long long off = rows_of(tok);
    load_k(off);
    load_v(off);
    for (; tok < stage_end; tok += kUnit) {
      const long long next = rows_of(tok + kUnit);
      if (off >= 0) {
        const float2 sc = s_scale[tok / g.page_size - first];
        // ---- scores ----
        float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ch = 0; ch < KL; ++ch) {
          const uint32_t lo[4] = {kr[ch][0].x, kr[ch][0].y, kr[ch][0].z, kr[ch][0].w};
          const uint32_t hi[4] = {kr[ch][1].x, kr[ch][1].y, kr[ch][1].z, kr[ch][1].w};
#pragma unroll
          for (int w = 0; w < 4; ++w)
            mma16816((w & 1) ? sb : sa, widen_lo(lo[w]), widen_lo(hi[w]), widen_hi(lo[w]), widen_hi(hi[w]), qf[ch * 4 + w][0], qf[ch * 4 + w][1]);
        }
        load_k(next);
        const float c0 = sc0 * sc.x, c1 = sc1 * sc.x;
        float s0 = (sa[0] + sb[0]) * c0, s1 = (sa[1] + sb[1]) * c1, s2 = (sa[2] + sb[2]) * c0, s3 = (sa[3] + sb[3]) * c1;
        if (tok + gq >= t_end) { s0 = -INFINITY; s1 = -INFINITY; }
        if (tok + gq + 8 >= t_end) { s2 = -INFINITY; s3 = -INFINITY; }
        // ---- running maximum and sum ----
        float mx0 = fmaxf(s0, s2), mx1 = fmaxf(s1, s3);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
        }
        const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
        const float b0 = n0 == -INFINITY ? 0.f : n0 - kPBits, b1 = n1 == -INFINITY ? 0.f : n1 - kPBits;
        float a0 = ex2f(m0 - kPBits - b0), a1 = ex2f(m1 - kPBits - b1);
        const float p0 = ex2f(s0 - b0), p1 = ex2f(s1 - b1), p2 = ex2f(s2 - b0), p3 = ex2f(s3 - b1);
        m0 = n0; m1 = n1;
        l0 = l0 * a0 + (p0 + p2);
        l1 = l1 * a1 + (p1 + p3);
        if (sc.y > r) {                   // a page with a larger V scale (the same for the whole warp)
          a0 *= r / sc.y; a1 *= r / sc.y;
          r = sc.y;
          inv_r = 1.f / r;
        }
        if (__any_sync(0xffffffffu, a0 != 1.f || a1 != 1.f)) {
#pragma unroll
          for (int j = 0; j < KS; ++j) { o[j][0] *= a0; o[j][1] *= a1; o[j][2] *= a0; o[j][3] *= a1; }
        }
        const float vs = sc.y * inv_r;
        const __half2 pa = __floats2half2_rn(p0 * vs, p1 * vs), pb = __floats2half2_rn(p2 * vs, p3 * vs);
        const uint32_t pt0 = transpose8x8(*reinterpret_cast<const uint32_t*>(&pa));
        const uint32_t pt1 = transpose8x8(*reinterpret_cast<const uint32_t*>(&pb));
        // ---- output ----
        const bool tail = tok + 16 > t_end;
#pragma unroll
        for (int hf = 0; hf < DH; ++hf) {
          if (tail) {                     // slots behind the last token may hold anything, NaN patterns included
            const uint4 z = make_uint4(0, 0, 0, 0);
            const int t = tok + 2 * tq;
            if (t >= t_end) vr[hf][0] = z;
            if (t + 1 >= t_end) vr[hf][1] = z;
            if (t + 8 >= t_end) vr[hf][2] = z;
            if (t + 9 >= t_end) vr[hf][3] = z;
          }
          const uint32_t wa[4] = {vr[hf][0].x, vr[hf][0].y, vr[hf][0].z, vr[hf][0].w}, wb[4] = {vr[hf][1].x, vr[hf][1].y, vr[hf][1].z, vr[hf][1].w};
          const uint32_t wc[4] = {vr[hf][2].x, vr[hf][2].y, vr[hf][2].z, vr[hf][2].w}, wd[4] = {vr[hf][3].x, vr[hf][3].y, vr[hf][3].z, vr[hf][3].w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x01 = __byte_perm(wa[w], wb[w], 0x5140), x23 = __byte_perm(wa[w], wb[w], 0x7362);
            const uint32_t y01 = __byte_perm(wc[w], wd[w], 0x5140), y23 = __byte_perm(wc[w], wd[w], 0x7362);
            mma16816(o[hf * 8 + 2 * w], widen_lo(x01), widen_hi(x01), widen_lo(y01), widen_hi(y01), pt0, pt1);
            mma16816(o[hf * 8 + 2 * w + 1], widen_lo(x23), widen_hi(x23), widen_lo(y23), widen_hi(y23), pt0, pt1);
          }
        }
        load_v(next);
      } else {
        load_k(next);
        load_v(next);
      }
      off = next;
    }
  }

  // ---- the four warps' states, through shared memory ----
#pragma unroll
  for (int x = 4; x < 32; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  if (gq == 0) {
    s_ml[warp][0][2 * tq] = m0; s_ml[warp][0][2 * tq + 1] = m1;
    s_ml[warp][1][2 * tq] = l0; s_ml[warp][1][2 * tq + 1] = l1;
  }
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    if (2 * tq + hh < G) {
      float* dst = s_acc + (warp * G + 2 * tq + hh) * D + 16 * gq;
#pragma unroll
      for (int hf = 0; hf < DH; ++hf)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<float4*>(dst + hf * 128 + 4 * w) = make_float4(o[hf * 8 + 2 * w][hh] * r, o[hf * 8 + 2 * w][2 + hh] * r,
                                                                          o[hf * 8 + 2 * w + 1][hh] * r, o[hf * 8 + 2 * w + 1][2 + hh] * r);
    }
  }
  __syncthreads();
  const long long stride = (long long)G * D + 16;
  float* part = p.part + (pair * p.num_splits) * stride;
  for (int i = tid; i < G * D / 4; i += kThreads) {
    const int j = i / (D / 4);
    float M = s_ml[0][0][j];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_ml[w][0][j]);
    float L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_ml[w][0][j] == -INFINITY ? 0.f : ex2f(s_ml[w][0][j] - M);
      const float4 v = reinterpret_cast<const float4*>(s_acc + w * G * D)[i];
      L += s_ml[w][1][j] * f;
      a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
    }
    if (pieces == 1) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
      reinterpret_cast<uint2*>(p.out + (lb * g.h_q + h * G) * D)[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    } else {
      reinterpret_cast<float4*>(part + split * stride)[i] = a;
      if (i % (D / 4) == 0) { part[split * stride + G * D + j] = M; part[split * stride + G * D + 8 + j] = L; }
    }
  }
  if (pieces == 1) return;

  // ---- the last piece to be finished joins all of them ----
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(p.counters + pair, 1) == pieces - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (tid == 0) p.counters[pair] = 0;
  for (int i = tid; i < G * D / 4; i += kThreads) {
    const int j = i / (D / 4);
    float M = -INFINITY, L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < pieces; ++s) M = fmaxf(M, __ldcg(part + s * stride + G * D + j));
#pragma unroll 8
    for (int s = 0; s < pieces; ++s) {
      const float ms = __ldcg(part + s * stride + G * D + j);
      const float f = ms == -INFINITY ? 0.f : ex2f(ms - M);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(part + s * stride) + i);
      L += __ldcg(part + s * stride + G * D + 8 + j) * f;
      a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
    reinterpret_cast<uint2*>(p.out + (lb * g.h_q + h * G) * D)[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// Pieces per pair: enough thread blocks for two rounds of a full GPU, none under 256 tokens.
int decode_splits(const PagedGeometry& g, int max_seq_len) {
  const long long cap = (long long)g.max_pages * g.page_size;
  const long long most = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  const long long pairs = (long long)g.n_layers * g.batch * g.h_kv;
  const long long slots = (long long)device_sms() * (g.head_dim == 128 ? 4 : 2);
  long long want = (2 * slots + pairs - 1) / pairs;
  const long long by_len = (most + 255) / 256;
  if (want > by_len) want = by_len;
  return (int)(want < 1 ? 1 : want > 128 ? 128 : want);
}

}  // namespace

size_t paged_decode_workspace_bytes(const PagedGeometry& g, int max_seq_len) {
  const size_t pairs = (size_t)g.n_layers * g.batch * g.h_kv, splits = decode_splits(g, max_seq_len);
  if (splits == 1) return 0;
  return pairs * splits * ((size_t)g.group * g.head_dim + 16) * 4 + pairs * 4;
}

cudaError_t launch_paged_decode(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  DecodeParams p{};
  p.g = g;
  p.q = (const uint16_t*)a.q;
  p.k_pages = (const uint8_t*)a.k_pages; p.v_pages = (const uint8_t*)a.v_pages;
  p.k_scale = a.k_scale; p.v_scale = a.v_scale;
  p.page_table = a.page_table; p.seq_len = a.seq_len;
  p.seq_len_offset = a.seq_len_offset;
  p.score_scale = a.softmax_scale * kLog2e;
  p.num_splits = decode_splits(g, a.max_seq_len);
  const long long pairs = (long long)g.n_layers * g.batch * g.h_kv;
  p.part = (float*)a.workspace;
  p.counters = (int*)(p.part + (size_t)pairs * p.num_splits * ((size_t)g.group * g.head_dim + 16));
  p.out = (uint16_t*)a.out;
  p.status = a.status;
  const long long grid = pairs * p.num_splits;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const size_t smem = (size_t)kWarps * g.group * g.head_dim * 4;
  auto launch = [&](auto kernel) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)grid, kThreads, smem, stream>>>(p);
    return cudaGetLastError();
  };
  return g.head_dim == 128 ? launch(paged_decode_kernel<128>) : launch(paged_decode_kernel<256>);
}

}  // namespace b200attn
