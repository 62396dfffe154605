// Attention of one query token per sequence over the paged FP8 cache: one scale per (page, kv head).
//
//   s_t = (q . k_t) * k_scale[page(t)] * softmax_scale * log2(e),   out = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m)
//
// Bound: HBM.  Every K and V byte of the attended tokens is read once and serves all G <= 8 query heads of its kv head.
//
// Two kernels (use_streamk says which, with the figures): one that starts and ends quickly for short caches and few of them,
// described here, and one that streams at the copy rate for everything else, described at its place.  One layer of one user on 512
// tokens takes 8 us; 64 layers of one on 8192 tokens 171 to 188 us issued from the host, by GPU and how warm it is (5.7 to 6.3 TB/s; 166 in a
// graph), 8 users on 65536 tokens with heads of 256 172 to 189 us (5.5 to 6.0 TB/s; 168 in a graph).
//
// A thread block of four warps takes a piece of one (layer, sequence, kv head) pair; a warp takes 16 tokens at a time,
// straight from global memory into registers in the layout that the tensor core wants, so there is nothing to fill, no
// barrier in the loop and no wait at its start.  (That is also why it stops short on long caches: each 16 tokens cost a warp 406
// instructions, and with 14 warps on an SM it reached 5.2 TB/s; the address arithmetic alone is what TMA takes over.)
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
// Sequences are cut into pieces over several thread blocks where there are few of them.  Each leaves (m, l, O) in the workspace and takes a
// ticket; the last one joins the pieces in order, so the result does not depend on who is last, and sets the counter
// back to zero.  Nobody waits for anybody.
#include "paged.cuh"
#include "streamk.cuh"

namespace b200attn {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16 * kWarps;        // tokens the block takes per round
constexpr int kMostPieces = 16;           // of a sequence
constexpr int kWhole = 256;               // sequences up to this many tokens are not cut into pieces
constexpr int kStage = 256;               // pages whose number and scales are in shared memory at a time
constexpr float kPBits = 15.f;            // p is held times 2^15
constexpr float kPUnit = 0x1p-15f;        // and sums leave the warp without that factor: times a loud V scale they could pass the largest float

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
  int* counters;                          // [pairs], used when pairs are cut into pieces (4 or more, so there are few pairs)
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
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
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

  pdl_wait();
  pdl_launch_dependents();
  const int len = paged_len(g, (long long)p.seq_len[b] + p.seq_len_offset, p.status, tid == 0 && split == 0 && h == 0 && layer == 0);
  // pieces: as many as the grid has room for, each a whole number of rounds
  const int rounds = (len + kUnit - 1) / kUnit;
  const int per = rounds * kUnit <= kWhole ? rounds : (rounds + p.num_splits - 1) / p.num_splits;
  const int pieces = per > 0 ? (rounds + per - 1) / per : 0;
  if (split >= pieces) {
    if (pieces == 0 && split == 0)        // no tokens: zeros
      for (int i = tid; i < G * D / 2; i += kThreads)
        reinterpret_cast<uint32_t*>(p.out + (lb * g.h_q + h * G) * D)[i] = 0u;
    return;
  }
  const int t_begin = split * per * kUnit, t_end = min(len, t_begin + per * kUnit);
  B200ATTN_CHECK(p.status, t_begin < t_end && layer < g.n_layers && pieces <= p.num_splits && pieces <= kMostPieces);

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
      B200ATTN_CHECK(p.status, t >= t_begin / g.page_size * g.page_size && t / g.page_size - first >= 0 && t / g.page_size - first < kStage);
      const int id = s_page[t / g.page_size - first];
      B200ATTN_CHECK(p.status, id < 0 || rows_exist(g, ((long long)id * g.h_kv + h) * g.page_size + t % g.page_size, 16, layer));
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
          const float louder = fmaxf(sc.y, kLeastScale);
          a0 *= r / louder; a1 *= r / louder;
          r = louder;
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
    s_ml[warp][1][2 * tq] = l0 * kPUnit; s_ml[warp][1][2 * tq + 1] = l1 * kPUnit;
  }
  auto sum_of = [&](float x) { return x * kPUnit * r; };
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    if (2 * tq + hh < G) {
      float* dst = s_acc + (warp * G + 2 * tq + hh) * D + 16 * gq;
#pragma unroll
      for (int hf = 0; hf < DH; ++hf)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<float4*>(dst + hf * 128 + 4 * w) = make_float4(sum_of(o[hf * 8 + 2 * w][hh]), sum_of(o[hf * 8 + 2 * w][2 + hh]),
                                                                          sum_of(o[hf * 8 + 2 * w + 1][hh]), sum_of(o[hf * 8 + 2 * w + 1][2 + hh]));
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
    float M = -INFINITY, L = 0.f, f[kMostPieces];
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < kMostPieces; ++s) {   // all loads of a group in flight together, whatever the number of pieces
      f[s] = s < pieces ? __ldcg(part + s * stride + G * D + j) : -INFINITY;
      M = fmaxf(M, f[s]);
    }
#pragma unroll
    for (int s0 = 0; s0 < kMostPieces; s0 += 8) {
      if (s0 >= pieces) break;
      float4 v[8];
      float l[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float* from = part + min(s0 + s, pieces - 1) * stride;
        v[s] = __ldcg(reinterpret_cast<const float4*>(from) + i);
        l[s] = __ldcg(from + G * D + 8 + j);
      }
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float w = f[s0 + s] == -INFINITY ? 0.f : ex2f(f[s0 + s] - M);
        L += l[s] * w;
        a.x += v[s].x * w; a.y += v[s].y * w; a.z += v[s].z * w; a.w += v[s].w * w;
      }
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
    reinterpret_cast<uint2*>(p.out + (lb * g.h_q + h * G) * D)[i] = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// ---------------------------------------------------------------------------------------------
// Much work: a persistent grid, the tiles of all pairs in one line divided evenly over it (stream-K), so that ragged batches of
// any shape fill the GPU and end together.  A producer warp streams K and V tiles of 64 tokens with TMA into a ring, one box
// per page (or piece of a page); four warps take 16 tokens of a tile each, as in the kernel above; an epilogue warp merges
// their states, and the CTA that holds a split pair's last piece collects the others' (tagged words, see streamk.cuh).
// ---------------------------------------------------------------------------------------------
constexpr int kTileT = 64;
constexpr int kThreadsP = (kConsumerWarps + 2) * 32;
constexpr int kDumps = 2;
constexpr int kMostStages = 5;            // tiles of the ring, if they fit
constexpr int kAhead = 8;                 // tiles whose pages and scales the producer looks up at a time

struct PagedMma {
  MmaParams m;                            // geometry (capacity = the table's), queries, lengths, workspace, output
  PagedGeometry g;
  const int* page_table;
  int page_shift;
};

template <int D, int MINB>
__global__ void __launch_bounds__(kThreadsP, MINB)
paged_streamk_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedMma pp) {
  constexpr int DH = D / 128;
  constexpr int KSTEPS = D / 16;
  constexpr int TILE_BYTES = kTileT * D;
  constexpr int DP = D + 4;
  const MmaParams& p = pp.m;
  const Geometry& g = p.g;
  const int G = g.group;
  const int stages = p.stages;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int gq = lane >> 2, tq = lane & 3;
  const uint32_t q_bytes = (uint32_t)G * D * 2;
  const int dump_warp_floats = G * DP;

  extern __shared__ __align__(16) uint8_t s_dyn[];
  const uint32_t raw_addr = smem_u32(s_dyn);
  uint8_t* smem = s_dyn + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sK = smem;
  uint8_t* sV = sK + (size_t)stages * TILE_BYTES;
  uint8_t* sQ = sV + (size_t)stages * TILE_BYTES;                                     // [2][G*D] bf16
  float* sDump = reinterpret_cast<float*>(sQ + 2 * q_bytes);                          // [2][4][G][DP]
  float* sML = sDump + kDumps * kConsumerWarps * dump_warp_floats;                    // [2][4][16]: m[8], l[8]
  float2* sScale = reinterpret_cast<float2*>(sML + kDumps * kConsumerWarps * 16);     // [stages][4]: K and V scale of 16 tokens; K < 0: no page
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + stages * 4);
  DeferredCombine* sComb = reinterpret_cast<DeferredCombine*>(bars + 2 * stages + 8);
  int* sFlags = reinterpret_cast<int*>(sComb + 1);                                    // [0] timed_out [1] queries [2] flags [3] tiles copied [4] fewest tiles of a CTA
  int* sLen = sFlags + 8;                                                             // [batch]
  int* sCum = sLen + g.batch;                                                         // [batch+1]
  volatile int* timed_out = sFlags;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8u * stages;
  const uint32_t qfull0 = empty0 + 8u * stages, qempty0 = qfull0 + 16u;
  const uint32_t dfull0 = qempty0 + 16u, dempty0 = dfull0 + 16u;

  if (tid == 32) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full0 + 8u * s, 1);
      mbar_init(empty0 + 8u * s, kConsumerWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(qfull0 + 8u * i, 1);
      mbar_init(qempty0 + 8u * i, kConsumerWarps);
      mbar_init(dfull0 + 8u * i, kConsumerWarps);
      mbar_init(dempty0 + 8u * i, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    sFlags[0] = 0; sFlags[1] = 0; sFlags[3] = 0;
    sComb->valid = 0;
  }
  if (warp == kProducerWarp && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  if (warp == 0) {   // lengths, and the tiles before each sequence
    pdl_wait();      // the kernel before this one has completed: lengths, cache and workspace are as it left them
    int before = 0, first_tiles = 0, longest = 0;
    bool any_empty = false, uniform = true;
    for (int b0 = 0; b0 < g.batch; b0 += 32) {
      const int b = b0 + lane;
      const int len = b < g.batch ? paged_len(pp.g, (long long)p.seq_len[b] + p.seq_len_offset, p.status, blockIdx.x == 0) : 0;
      const int n = (len + kTileT - 1) / kTileT;
      if (b0 == 0) first_tiles = __shfl_sync(0xffffffffu, n, 0);
      longest = max(longest, __reduce_max_sync(0xffffffffu, n));
      any_empty |= __any_sync(0xffffffffu, b < g.batch && n == 0);
      uniform &= __all_sync(0xffffffffu, b >= g.batch || n == first_tiles);
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += t;
      }
      if (b < g.batch) { sLen[b] = len; sCum[b] = before + inc - n; }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) { sCum[g.batch] = before; sFlags[2] = (any_empty ? 1 : 0) | (uniform ? 2 : 0); sFlags[4] = max(1, (int)ceilf(sqrtf((float)longest))); }
  } else {
    pdl_wait();
  }
  __syncthreads();
  if (tid == 0) pdl_launch_dependents();

  if (sFlags[2] & 1) {   // sequences without tokens: zeros
    const long long rows = (long long)g.n_layers * g.batch;
    for (long long r = blockIdx.x; r < rows; r += gridDim.x)
      if (sLen[r % g.batch] == 0)
        for (int i = tid; i < g.h_q * D / 2; i += kThreadsP) reinterpret_cast<uint32_t*>(p.out + r * g.h_q * D)[i] = 0u;
  }
  const long long total = (long long)sCum[g.batch] * g.h_kv * g.n_layers;
  // A piece takes time with its tiles, a join with its pieces: at least the root of the longest sequence's tiles per CTA
  // (one pair of 8192 tokens cut into 128 pieces: 92 us).
  const long long most_ctas = max(1LL, total / sFlags[4]);
  int n_eff;
  long long r0, r1;
  cta_range(total, (int)min((long long)gridDim.x, most_ctas), (int)blockIdx.x, (sFlags[2] & 2) ? sCum[1] - sCum[0] : 0, n_eff, r0, r1);
  const bool has_work = r0 < r1;

  if (warp == kProducerWarp) {
    if (has_work) {
      // Lane 4 k + i looks up the page and the scales of tokens 16 i .. of the k-th tile of the next kAhead; the lane of a box's
      // first 16 tokens (a box: a page, or the 64 tokens of the tile that a larger page holds) then issues its copies.
      const uint64_t policy = l2_policy_evict_first();
      const int box_rows = min(pp.g.page_size, kTileT), n_it = (int)(r1 - r0);
      int id = -1, row = 0, layer = 0, seg_pair = -1, pair = 0, seg = 0;
      float2 sc = make_float2(0.f, 0.f);
      auto look_up = [&](int it0, int& id_, int& row_, int& layer_, int& pair_, float2& sc_) {
        id_ = -1; row_ = 0; sc_ = make_float2(0.f, 0.f); layer_ = 0; pair_ = 0;
        const int it = it0 + (lane >> 2);
        if (it >= n_it) return;
        const Cursor c = locate(r0 + it, sCum, sLen, g.batch, g.h_kv);
        layer_ = c.layer;
        pair_ = (c.layer * g.batch + c.b) * g.h_kv + c.h;
        const int tok = c.tile * kTileT + (lane & 3) * 16;
        if (tok >= c.len_b) return;
        B200ATTN_CHECK(p.status, c.b >= 0 && c.b < g.batch && tok >= 0 && (tok >> pp.page_shift) < pp.g.max_pages);
        const int page = ld(pp.page_table + (long long)c.b * pp.g.max_pages + (tok >> pp.page_shift));
        if (page < 0 || page >= pp.g.n_pages) {
          atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE);
          sc_.x = -1.f;
          return;
        }
        id_ = page;
        row_ = ((page * g.h_kv + c.h) << pp.page_shift) + (tok & (pp.g.page_size - 1));
        const long long si = ((long long)c.layer * pp.g.n_pages + page) * g.h_kv + c.h;
        sc_ = make_float2(ld(p.k_scale + si), ld(p.v_scale + si));
      };
      int id2, row2, layer2, pair2_;
      float2 sc2;
      look_up(0, id, row, layer, pair, sc);
      bool ok = true;
      int s = 0, lap = 0;                   // slot of the ring, times around it
      for (int it0 = 0; it0 < n_it && ok; it0 += kAhead) {
        look_up(it0 + kAhead, id2, row2, layer2, pair2_, sc2);
        for (int k = 0; k < kAhead && it0 + k < n_it; ++k) {
          const int it = it0 + k;
          const int cur_pair = __shfl_sync(0xffffffffu, pair, 4 * k);
          if (cur_pair != seg_pair) {   // the G query rows of this pair
            const int qb = seg & 1;
            if (seg >= 2) ok = mbar_wait(qempty0 + 8u * qb, ((seg >> 1) - 1) & 1, timed_out, p.status);
            __syncwarp();
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(qfull0 + 8u * qb, q_bytes);
              const int lb = cur_pair / g.h_kv;
              bulk_load(smem_u32(sQ + qb * q_bytes), p.q + ((long long)lb * g.h_q + (cur_pair - lb * g.h_kv) * G) * D, q_bytes, qfull0 + 8u * qb);
            }
            seg_pair = cur_pair;
            ++seg;
          }
          if (lap) ok = mbar_wait(empty0 + 8u * s, (lap - 1) & 1, timed_out, p.status);
          __syncwarp();
          if (!ok) break;
          const uint32_t fb = full0 + 8u * s;
          const bool mine = (lane >> 2) == k;
          if (mine) sScale[s * 4 + (lane & 3)] = sc;
          const bool box = mine && id >= 0 && ((lane & 3) * 16) % box_rows == 0;
          const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, box));
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(fb, 2u * boxes * box_rows * D);
          __syncwarp();
          if (box) {
            B200ATTN_CHECK(p.status, rows_exist(pp.g, row, box_rows, layer) && s >= 0 && s < stages && (lane & 3) * 16 + box_rows <= kTileT);
#pragma unroll
            for (int hf = 0; hf < DH; ++hf) {
              const uint32_t off = (uint32_t)s * TILE_BYTES + hf * kTileT * 128 + (lane & 3) * 16 * 128;
              tma_load_3d_hint(smem_u32(sK) + off, &kmap, hf * 128, row, layer, fb, policy);
              tma_load_3d_hint(smem_u32(sV) + off, &vmap, hf * 128, row, layer, fb, policy);
            }
          }
          if (lane == 0) { sFlags[3] = it + 1; sFlags[1] = seg; }   // for the drain after a wait that ran out
          if (++s == stages) { s = 0; ++lap; }
        }
        id = id2; row = row2; layer = layer2; pair = pair2_; sc = sc2;
      }
    }
  } else if (warp == kEpilogueWarp) {
    if (has_work)
      epilogue_warp<D, kDumps, kConsumerWarps, false, true>(p, lane, r0, r1, total, n_eff, sCum, sLen, sDump, sML, dfull0, dempty0, timed_out,
                                                           nullptr, sComb, 0);
  } else if (has_work) {
    Cursor c = locate(r0, sCum, sLen, g.batch, g.h_kv);
    long long cur = r0;
    int s = 0, lap = 0, seg = 0;
    const uint32_t sK_addr = smem_u32(sK), sV_addr = smem_u32(sV);
    const int row_lo = warp * 16 + gq;
    while (cur < r1) {
      const long long pair_end = cur - c.tile + c.tiles_b, seg_end = pair_end < r1 ? pair_end : r1;
      const int ntiles = (int)(seg_end - cur), qb = seg & 1;
      // ---- query fragments: head gq, dims hf * 128 + 32 tq + 4 ks ..; each head scaled by a power of two into f16's range ----
      uint32_t qf[KSTEPS][2];
      float sc0, sc1;
      {
        const bool qok = mbar_wait(qfull0 + 8u * qb, (seg >> 1) & 1, timed_out, p.status);
        float qv[DH][32];
        float amax = 0.f;
#pragma unroll
        for (int hf = 0; hf < DH; ++hf)
#pragma unroll
          for (int v4 = 0; v4 < 4; ++v4) {
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (gq < G && qok) raw = lds128(smem_u32(sQ + qb * q_bytes) + (gq * D + 32 * tq) * 2 + hf * 256 + v4 * 16);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              qv[hf][v4 * 8 + 2 * i] = bf16_bits_to_float(w[i] & 0xFFFFu);
              qv[hf][v4 * 8 + 2 * i + 1] = bf16_bits_to_float(w[i] >> 16);
              amax = fmaxf(amax, fmaxf(fabsf(qv[hf][v4 * 8 + 2 * i]), fabsf(qv[hf][v4 * 8 + 2 * i + 1])));
            }
          }
        __syncwarp();
        if (lane == 0) mbar_arrive(qempty0 + 8u * qb);
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int ex = (int)((__float_as_uint(amax) >> 23) & 0xFF);
        ex = ex < 1 ? 1 : (ex > 253 ? 253 : ex);
        const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
        for (int hf = 0; hf < DH; ++hf)
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const __half2 b0 = __floats2half2_rn(qv[hf][4 * w] * down, qv[hf][4 * w + 1] * down);
            const __half2 b1 = __floats2half2_rn(qv[hf][4 * w + 2] * down, qv[hf][4 * w + 3] * down);
            qf[hf * 8 + w][0] = *reinterpret_cast<const uint32_t*>(&b0);
            qf[hf * 8 + w][1] = *reinterpret_cast<const uint32_t*>(&b1);
          }
        const float mult = up * p.score_scale;
        sc0 = __shfl_sync(0xffffffffu, mult, 8 * tq);
        sc1 = __shfl_sync(0xffffffffu, mult, 8 * tq + 4);
      }
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, r = 0.f, inv_r = 0.f;
      float o[KSTEPS][4];
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f; }

      for (int ti = 0; ti < ntiles; ++ti) {
        const bool ok = mbar_wait(full0 + 8u * s, lap & 1, timed_out, p.status);
        const int tok0 = (c.tile + ti) * kTileT + warp * 16;
        const float2 sc = sScale[s * 4 + warp];
        if (ok && tok0 < c.len_b && sc.x >= 0.f) {
          float sacc[4] = {0.f, 0.f, 0.f, 0.f}, sacc2[4] = {0.f, 0.f, 0.f, 0.f};
          const uint32_t kt = sK_addr + s * TILE_BYTES;
#pragma unroll
          for (int hf = 0; hf < DH; ++hf)
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              const uint32_t off = hf * kTileT * 128 + (((2 * tq + ch) ^ gq) << 4);
              const uint4 klo = lds128(kt + off + row_lo * 128), khi = lds128(kt + off + (row_lo + 8) * 128);
              const uint32_t wl[4] = {klo.x, klo.y, klo.z, klo.w}, wh[4] = {khi.x, khi.y, khi.z, khi.w};
#pragma unroll
              for (int w = 0; w < 4; ++w)
                mma_f16((w & 1) ? sacc2 : sacc, cvt_lo(wl[w]), cvt_lo(wh[w]), cvt_hi(wl[w]), cvt_hi(wh[w]), qf[hf * 8 + ch * 4 + w][0], qf[hf * 8 + ch * 4 + w][1]);
            }
          const float c0 = sc0 * sc.x, c1 = sc1 * sc.x;
          float s0 = (sacc[0] + sacc2[0]) * c0, s1 = (sacc[1] + sacc2[1]) * c1, s2 = (sacc[2] + sacc2[2]) * c0, s3 = (sacc[3] + sacc2[3]) * c1;
          if (tok0 + gq >= c.len_b) { s0 = -INFINITY; s1 = -INFINITY; }
          if (tok0 + gq + 8 >= c.len_b) { s2 = -INFINITY; s3 = -INFINITY; }
          float mx0 = fmaxf(s0, s2), mx1 = fmaxf(s1, s3);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
          }
          const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
          const float b0 = n0 == -INFINITY ? 0.f : n0 - kPBits, b1 = n1 == -INFINITY ? 0.f : n1 - kPBits;
          float a0 = ex2(m0 - kPBits - b0), a1 = ex2(m1 - kPBits - b1);
          const float p0 = ex2(s0 - b0), p1 = ex2(s1 - b1), p2 = ex2(s2 - b0), p3 = ex2(s3 - b1);
          m0 = n0; m1 = n1;
          l0 = l0 * a0 + (p0 + p2);
          l1 = l1 * a1 + (p1 + p3);
          if (sc.y > r) {                 // a page with a larger V scale (the same for the whole warp)
            const float louder = fmaxf(sc.y, kLeastScale);
            a0 *= r / louder; a1 *= r / louder;
            r = louder;
            inv_r = 1.f / r;
          }
          if (__any_sync(0xffffffffu, a0 != 1.f || a1 != 1.f)) {
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j) { o[j][0] *= a0; o[j][1] *= a1; o[j][2] *= a0; o[j][3] *= a1; }
          }
          const float vs = sc.y * inv_r;
          const __half2 pa = __floats2half2_rn(p0 * vs, p1 * vs), pb = __floats2half2_rn(p2 * vs, p3 * vs);
          const uint32_t pb0 = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&pa)), pb1 = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&pb));
          const uint32_t vt = sV_addr + s * TILE_BYTES;
          const int vr = warp * 16 + 2 * tq;
          const bool tail = tok0 + 16 > c.len_b;
#pragma unroll
          for (int hf = 0; hf < DH; ++hf) {
            const uint32_t vb = vt + hf * kTileT * 128;
            uint4 va = lds128(vb + vr * 128 + ((gq ^ (2 * tq)) << 4)), vbb = lds128(vb + (vr + 1) * 128 + ((gq ^ (2 * tq + 1)) << 4));
            uint4 vc = lds128(vb + (vr + 8) * 128 + ((gq ^ (2 * tq)) << 4)), vd = lds128(vb + (vr + 9) * 128 + ((gq ^ (2 * tq + 1)) << 4));
            if (tail) {                   // slots behind the last token may hold anything, NaN patterns included
              const int tv = tok0 + 2 * tq;
              const uint4 z = make_uint4(0, 0, 0, 0);
              if (tv >= c.len_b) va = z;
              if (tv + 1 >= c.len_b) vbb = z;
              if (tv + 8 >= c.len_b) vc = z;
              if (tv + 9 >= c.len_b) vd = z;
            }
            const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vbb.x, vbb.y, vbb.z, vbb.w};
            const uint32_t wc[4] = {vc.x, vc.y, vc.z, vc.w}, wd[4] = {vd.x, vd.y, vd.z, vd.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t x01 = prmt(wa[w], wb[w], 0x5140), x23 = prmt(wa[w], wb[w], 0x7362), y01 = prmt(wc[w], wd[w], 0x5140), y23 = prmt(wc[w], wd[w], 0x7362);
              mma_f16(o[hf * 8 + 2 * w], cvt_lo(x01), cvt_hi(x01), cvt_lo(y01), cvt_hi(y01), pb0, pb1);
              mma_f16(o[hf * 8 + 2 * w + 1], cvt_lo(x23), cvt_hi(x23), cvt_lo(y23), cvt_hi(y23), pb0, pb1);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8u * s);
        if (++s == stages) { s = 0; ++lap; }
      }
      // ---- end of the segment: the warp's state to the epilogue warp ----
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      const int db = seg % kDumps;
      if (seg < kDumps || mbar_wait(dempty0 + 8u * db, ((seg / kDumps) - 1) & 1, timed_out, p.status)) {
        float* ml = sML + (db * kConsumerWarps + warp) * 16;
        if (gq == 0) {
          ml[2 * tq] = m0; ml[2 * tq + 1] = m1;
          ml[8 + 2 * tq] = l0 * kPUnit; ml[8 + 2 * tq + 1] = l1 * kPUnit;
        }
        const uint32_t dbase = smem_u32(sDump + (db * kConsumerWarps + warp) * dump_warp_floats);
        auto sum_of = [&](float x) { return x * kPUnit * r; };
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j) {   // regs 0, 1: dim (j >> 3) * 128 + 16 gq + 2 (j & 7) of heads 2 tq, 2 tq + 1; regs 2, 3: that dim + 1
          const int u = (j >> 3) * 64 + 8 * gq + (j & 7);
          const uint32_t pos8 = 8u * (uint32_t)((u & ~7) | ((j & 7) ^ gq));
          if (2 * tq < G) sts64(dbase + 2 * tq * DP * 4 + pos8, sum_of(o[j][0]), sum_of(o[j][2]));
          if (2 * tq + 1 < G) sts64(dbase + (2 * tq + 1) * DP * 4 + pos8, sum_of(o[j][1]), sum_of(o[j][3]));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(dfull0 + 8u * db);
      ++seg;
      cur = seg_end;
      if (cur < r1) next_pair(c, sCum, sLen, g.batch, g.h_kv);
    }
  }
  __syncthreads();
  if (sFlags[0] && tid == kConsumerThreads) {
    // A wait ran out.  Copies already issued still land in this CTA's shared memory: wait for them (bounded).
    const int n_it = sFlags[3], segs = sFlags[1];
    for (int s = 0; s < stages && s < n_it; ++s) {
      const int last = ((n_it - 1 - s) / stages) * stages + s;
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(full0 + 8u * s, (last / stages) & 1) && global_timer_ns() - t0 < kWaitBudgetNs) {}
    }
    for (int qb = 0; qb < 2 && qb < segs; ++qb) {
      const int last = ((segs - 1 - qb) / 2) * 2 + qb;
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(qfull0 + 8u * qb, (last >> 1) & 1) && global_timer_ns() - t0 < kWaitBudgetNs) {}
    }
  }
  if (sComb->valid && !sFlags[0]) combine_deferred<D>(combine_args_of(p, nullptr, 0), *sComb, warp, kThreadsP / 32, lane);
}

size_t streamk_smem(const PagedGeometry& g, int stages) {
  size_t b = 1024;
  b += (size_t)2 * stages * kTileT * g.head_dim;
  b += (size_t)2 * g.group * g.head_dim * 2;
  b += (size_t)kDumps * kConsumerWarps * g.group * (g.head_dim + 4) * 4;
  b += (size_t)kDumps * kConsumerWarps * 16 * 4;
  b += (size_t)stages * 4 * 8;
  b += (size_t)(2 * stages + 8) * 8;
  b += sizeof(DeferredCombine) + 32;
  b += (size_t)(2 * g.batch + 1) * 4;
  return (b + 15) & ~(size_t)15;
}
// CTAs per SM of the persistent grid, and the ring with which they fit.  Heads of 128, 32 sequences to 16384 tokens / 64 layers x 8192: three
// CTAs with 3 tiles 101 / 177 us, two with 3, 4, 5, 6 tiles 93 / 172, 89 / 167, 89 / 166, 89 / 166; heads of 256, 8 x 65536: one CTA
// with 3, 4, 5 tiles 174, 168, 168, two with 2 tiles 206.
int streamk_ctas_per_sm(const PagedGeometry& g) { return g.head_dim == 128 ? 2 : 1; }
int streamk_stages(const PagedGeometry& g) {
  int n = kMostStages;
  while (n > 2 && (streamk_smem(g, n) + 1024) * streamk_ctas_per_sm(g) > 227 * 1024) --n;
  return n;
}

// Longest sequence a call can meet, as far as the host knows.
long long most_tokens(const PagedGeometry& g, int max_seq_len) {
  const long long cap = (long long)g.max_pages * g.page_size;
  return max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
}

// Which kernel: the register kernel starts and ends faster, the stream-K kernel streams faster and balances.  Heads of 128,
// register / stream-K, us: 256 tokens, 8 pairs 6.4 / 8.5, 1024 pairs 20 / 23; 512 tokens, 256 pairs 13.9 / 12.5, 1024 pairs 32 / 34;
// 1024 tokens, 8 pairs 9.7 / 10.2, 256 pairs 23 / 18, 1024 pairs 55 / 55; 2048 tokens, 64 pairs 15.3 / 15.7, 1024 pairs 100 / 93; 8192
// tokens, 8 pairs 17 / 20, 64 pairs 33 / 31, 1024 pairs 392 / 358.  Heads of 256: 512 tokens, 512 pairs 34 / 37; 1024 tokens, 128 pairs
// 25 / 20; 2048 tokens, 32 pairs 16 / 18; 8192 tokens, 32 pairs 34 / 34, 128 pairs 173 / 98.
bool use_streamk(const PagedGeometry& g, int max_seq_len) {
  if (g.batch > kMaxBatchMma || (long long)g.n_pages * g.h_kv * g.page_size > 0x7fffffffLL) return false;
  const long long most = most_tokens(g, max_seq_len), pairs = (long long)g.n_layers * g.batch * g.h_kv;
  return most > 768 && most * g.head_dim * pairs > (1LL << 24);
}

// Register kernel: pieces per pair.  Joining costs about 4 us and grows with their number, so few pairs are cut into up to 16,
// and many pairs not at all (8 pairs of 512 tokens: 8 pieces 8.1 us, whole 9.6; of 8192: 32 pieces 16 us, 128 pieces 39;
// 256 pairs of 512: 3 pieces 21 us, whole 14).
int decode_splits(const PagedGeometry& g, int max_seq_len) {
  const long long most = most_tokens(g, max_seq_len), pairs = (long long)g.n_layers * g.batch * g.h_kv;
  const long long slots = (long long)device_sms() * (g.head_dim == 128 ? 4 : 2);
  long long n = slots / pairs;
  const long long by_len = (most + kUnit - 1) / kUnit;
  n = n < by_len ? n : by_len;
  return most <= kWhole || n < 4 ? 1 : n > kMostPieces ? kMostPieces : (int)n;
}

}  // namespace

size_t paged_decode_workspace_bytes() {
  // register kernel: partial states of at most every block slot of the device
  return paged_partials_offset() + (size_t)device_sms() * 4 * (8 * 128 + 16) * 4;
}

namespace {

cudaError_t launch_paged_streamk(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  Geometry cache{};
  cache.n_layers = g.n_layers; cache.batch = g.n_pages; cache.h_kv = g.h_kv; cache.capacity = g.page_size; cache.head_dim = g.head_dim;
  const int box = g.page_size < kTileT ? g.page_size : kTileT;
  CUtensorMap kmap, vmap;
  if (!encode_cache_map(&kmap, a.k_pages, cache, g.k_layer_stride, box) || !encode_cache_map(&vmap, a.v_pages, cache, g.v_layer_stride, box))
    return cudaErrorInvalidValue;
  PagedMma p{};
  p.g = g;
  p.page_table = a.page_table;
  p.page_shift = g.page_size == 16 ? 4 : g.page_size == 32 ? 5 : g.page_size == 64 ? 6 : 7;
  MmaParams& m = p.m;
  m.g.n_layers = g.n_layers; m.g.batch = g.batch; m.g.h_q = g.h_q; m.g.h_kv = g.h_kv; m.g.head_dim = g.head_dim; m.g.group = g.group;
  m.g.capacity = g.max_pages * g.page_size;
  m.q = (const uint16_t*)a.q;
  m.k_scale = a.k_scale; m.v_scale = a.v_scale;
  m.seq_len = a.seq_len;
  m.seq_len_offset = a.seq_len_offset;
  m.score_scale = a.softmax_scale * kLog2e;
  m.ws_pkt = paged_words(a.workspace);
  m.out = (uint16_t*)a.out;
  m.out_hq_total = g.h_q;
  m.status = a.status;
  m.stages = streamk_stages(g);
  const int n = streamk_ctas_per_sm(g) * device_sms();
  const size_t smem = streamk_smem(g, m.stages);
  auto launch = [&](auto kernel) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, n, kThreadsP, smem, stream, kmap, vmap, p);
  };
  return g.head_dim == 128 ? launch(paged_streamk_kernel<128, 2>) : launch(paged_streamk_kernel<256, 1>);
}

}  // namespace

cudaError_t launch_paged_decode(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  if (use_streamk(g, a.max_seq_len)) return launch_paged_streamk(g, a, stream);
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
  p.part = paged_partials(a.workspace);
  p.counters = paged_counters(a.workspace);
  p.out = (uint16_t*)a.out;
  p.status = a.status;
  const long long grid = pairs * p.num_splits;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const size_t smem = (size_t)kWarps * g.group * g.head_dim * 4;   // at most 32 KB
  return g.head_dim == 128 ? launch_pdl(paged_decode_kernel<128>, (int)grid, kThreads, smem, stream, p)
                           : launch_pdl(paged_decode_kernel<256>, (int)grid, kThreads, smem, stream, p);
}

}  // namespace b200attn
