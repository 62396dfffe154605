// Attention of a few query tokens per sequence over the paged FP8 cache (guessed tokens to be verified, short continuations).
//
// Bound: issue slots and HBM together.  The K and V bytes are read once and serve all query rows of a tile, up to 8 NT = 16 rows
// (tokens x heads of the kv head); 16 tokens of keys cost a warp about 1,000 cycles of its quarter of an SM, the copy rate would
// allow 720.  Against the kernel for tiles of 128 rows: 8 sequences x 2 tokens on 12288 to 16384 keys, 40 / 8 heads of 128, 62 us
// (4.2 TB/s) and 94 us; on 768 to 1024 keys 14.6 and 17.3 us; heads of 256 (24 / 4) 61 and 76, 15.5 and 25 us.  With 32 rows a
// tile (NT = 4) it was the slower one, 39 us against 34 for 4 tokens x 5 heads on about 3500 keys, so it stops at 16.
//
// A thread block of four warps takes a tile of query rows and a piece of the keys.  Every warp is on its own: it has a ring of
// 16-token slots that its lane 0 fills by TMA (one box of 16 rows each for K and V and 128-byte half, so a page is a whole number
// of boxes) and consumes them with mma.m16n8k16, NT column tiles of 8 query rows each:
//   S^T[16 tokens x 8 rows] = K q^T with K widened to f16 (exact),   O^T[D x 8 rows] += V^T P^T with P^T from a movmatrix transpose.
// There is no barrier between the warps until their states are joined in shared memory, and a refill only waits for its own warp.
// The query fragments are the same for all warps and stay in shared memory; O takes up to 128 registers.  Pieces of the keys are joined by the last block to finish, in order, as for one query token.
// Precision: as for one query token (q in f16 scaled by a power of two per row, p * 2^15 in f16, fp32 sums and accumulators).
#include "paged.cuh"
#include "streamk.cuh"

namespace b200attn {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kRowsU = 16;                // tokens of a unit
constexpr float kPBits = 15.f;            // p is held times 2^15
constexpr float kPUnit = 0x1p-15f;        // and sums leave the warp without that factor: times a loud V scale they could pass the largest float
constexpr int kTilesN = 2, kFewRows = 8 * kTilesN;   // column tiles, query rows of a tile
constexpr int kMostPieces = 16;           // of the keys
constexpr int kLeastUnits = 16;           // units of a piece, at least (8: 8 sequences of 256 keys 9.5 us for 8.0; 32: 1024 keys 14 us for 11)

template <int D, int NT>
struct FewPlan {
  static constexpr int DH = D / 128, SLOT = 2 * kRowsU * D;             // bytes of a slot: K, then V
  static constexpr int SLOTS = D == 128 ? 4 : 3;                        // 64 KB (96 KB with heads of 256) in flight per block are plenty
  static constexpr int BLOCKS = D == 128 ? 3 : 2;                       // per SM (two: 8 x 2 tokens on 16384 keys 75 us, three 62)
  static constexpr int COLS = 8 * NT;
  static constexpr int RING = kWarps * SLOTS * SLOT;
  static constexpr int QF = NT * (D / 16) * 32 * 8;
  static constexpr int SMEM = 1024 + RING + QF;
  static_assert(kWarps * COLS * D * 4 <= RING, "the warps' states are joined where the ring was");
};

struct FewParams {
  PagedGeometry g;
  const uint16_t* q;
  const float *k_scale, *v_scale;
  const int *page_table, *seq_len, *q_start;
  int n_tokens, causal, page_shift, splits, tiles, per_tile;   // per_tile: query tokens of a tile
  float score_scale;
  float* part;                            // [block][piece][COLS * D + 2 * COLS]: O, m, l
  int* counters;                          // [block]
  uint16_t* out;
  int* status;
};

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, (FewPlan<D, NT>::BLOCKS))
paged_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const FewParams p) {
  using P = FewPlan<D, NT>;
  constexpr int DH = P::DH, KS = D / 16, S = P::SLOTS, COLS = P::COLS;
  const PagedGeometry& g = p.g;
  const int G = g.group, tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int gq = lane >> 2, tq = lane & 3;

  extern __shared__ uint8_t s_dyn[];
  __shared__ __align__(8) uint64_t s_bar[kWarps][S];
  __shared__ float2 s_sc[kWarps][S];      // K and V scale of the slot's tokens; K < 0: no page
  __shared__ float s_mul[COLS], s_ml[kWarps][2][COLS];
  __shared__ int s_vis[COLS], s_info[8];  // sequence, tile of it, first row, rows, length, timed out, last
  const uint32_t ring = (smem_u32(s_dyn) + 1023u) & ~1023u;
  uint8_t* ring_ptr = s_dyn + (ring - smem_u32(s_dyn));
  uint2* s_qf = reinterpret_cast<uint2*>(ring_ptr + P::RING);             // [NT][KS][32]
  volatile int* timed_out = s_info + 5;

  // ---- which tile: piece fastest, then head, layer, query tile ----
  const int piece = (int)(blockIdx.x % p.splits);
  int rest = blockIdx.x / p.splits;
  const int h = rest % g.h_kv;
  rest /= g.h_kv;
  const int layer = rest % g.n_layers, number = rest / g.n_layers;
  if (lane < S) mbar_init(smem_u32(&s_bar[warp][lane]), 1);
  if (tid < 8) s_info[tid] = tid == 0 ? -1 : 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  pdl_wait();
  __syncthreads();
  if (warp == 0) {
    int before = 0;
    for (int b0 = 0; b0 < g.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0, q0 = 0, nq = 0, raw_len = 0;
      if (b < g.batch) {
        q0 = p.q_start[b];
        const int end = p.q_start[b + 1];
        nq = end - q0;
        raw_len = p.seq_len[b];
        if (range_fits(q0, end, p.n_tokens, p.status, blockIdx.x == 0) && nq > 0) n = (nq + p.per_tile - 1) / p.per_tile;
      }
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += t;
      }
      const int start = before + inc - n;
      if (n > 0 && number >= start && number < start + n) { s_info[0] = b; s_info[1] = number - start; s_info[2] = q0; s_info[3] = nq; s_info[4] = raw_len; }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > number && blockIdx.x != 0) break;         // the first block has looked at every sequence
    }
  }
  __syncthreads();
  pdl_launch_dependents();
  const int b = s_info[0];
  if (b < 0) return;                      // the grid is an upper bound
  const int first_tok = s_info[1] * p.per_tile, ntok = min(p.per_tile, s_info[3] - first_tok);
  const int len = paged_len(g, s_info[4], p.status, tid == 0 && layer == 0 && h == 0 && piece == 0);
  const int hidden = len - s_info[3] + first_tok + 1;                     // causal: token t of the tile sees the first hidden + t keys
  const int visible = p.causal ? min(len, max(0, hidden + ntok - 1)) : len;
  const int units = (visible + kRowsU - 1) / kRowsU;
  const int per = ((units + p.splits - 1) / p.splits + kWarps - 1) / kWarps * kWarps;
  const int pieces = per > 0 ? (units + per - 1) / per : 0;
  const long long row0 = ((long long)layer * p.n_tokens + s_info[2] + first_tok) * g.h_q + h * G;   // of (token 0, head 0)
  if (piece >= pieces) {
    if (pieces == 0 && piece == 0)        // nothing to see: zeros
      for (int i = tid; i < ntok * G * (D / 8); i += kThreads) {
        const int row = i / (D / 8);
        reinterpret_cast<uint4*>(p.out + (row0 + (long long)(row / G) * g.h_q + row % G) * D)[i % (D / 8)] = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  B200ATTN_CHECK(p.status, first_tok >= 0 && ntok > 0 && ntok * G <= COLS && layer < g.n_layers && s_info[2] + first_tok + ntok <= p.n_tokens &&
                               pieces <= p.splits && pieces <= kMostPieces && visible <= g.max_pages * g.page_size);
  const int u0 = piece * per + warp, u1 = min(units, piece * per + per);
  const int n = u1 > u0 ? (u1 - u0 + kWarps - 1) / kWarps : 0;            // units of this warp: u0, u0 + kWarps, ..

  // ---- the ring ----
  const uint32_t my_ring = ring + warp * (S * P::SLOT), my_bar = smem_u32(&s_bar[warp][0]);
  auto look_up = [&](int i0, int& row, float2& sc) {   // lane: unit i0 + lane; row < 0: nothing to copy
    row = -1;
    sc = make_float2(-1.f, 0.f);
    if (i0 + lane >= n) return;
    const int tok = (u0 + (i0 + lane) * kWarps) * kRowsU;
    B200ATTN_CHECK(p.status, tok < visible && (tok >> p.page_shift) < g.max_pages);
    const int page = ld(p.page_table + (long long)b * g.max_pages + (tok >> p.page_shift));
    if (page < 0 || page >= g.n_pages) { atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE); return; }
    row = ((page * g.h_kv + h) << p.page_shift) + (tok & (g.page_size - 1));
    const long long si = ((long long)layer * g.n_pages + page) * g.h_kv + h;
    sc = make_float2(ld(p.k_scale + si), ld(p.v_scale + si));
  };
  int row, next_row;
  float2 sc, next_sc;
  look_up(0, row, sc);
  look_up(32, next_row, next_sc);
  auto issue = [&](int i) {
    if (i > 0 && (i & 31) == 0) {
      row = next_row; sc = next_sc;
      look_up(i + 32, next_row, next_sc);
    }
    const int s = i % S;
    if (lane == (i & 31)) {
      s_sc[warp][s] = sc;
      const uint32_t bar = my_bar + 8 * s, dst = my_ring + s * P::SLOT;
      if (row >= 0) {
        B200ATTN_CHECK(p.status, rows_exist(g, row, kRowsU, layer));
        mbar_arrive_expect_tx(bar, P::SLOT);
#pragma unroll
        for (int hf = 0; hf < DH; ++hf) {
          tma_load_3d(dst + hf * (kRowsU * 128), &kmap, hf * 128, row, layer, bar);
          tma_load_3d(dst + kRowsU * D + hf * (kRowsU * 128), &vmap, hf * 128, row, layer, bar);
        }
      } else {
        mbar_arrive(bar);
      }
    }
    __syncwarp();
  };
  int issued = 0;
  for (; issued < S && issued < n; ++issued) issue(issued);

  // ---- query fragments: column 8 nt + gq, dims hf * 128 + 32 tq + 4 w .. + 3 ----
  for (int nt = warp; nt < NT; nt += kWarps) {
    const int col = nt * 8 + gq, tok = col / G;
    const bool real = tok < ntok;         // per_tile * G <= COLS
    float x[DH][32], amax = 0.f;
#pragma unroll
    for (int hf = 0; hf < DH; ++hf)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (real) raw = ld(reinterpret_cast<const uint4*>(p.q + (row0 + (long long)tok * g.h_q + col % G) * D + hf * 128 + 32 * tq + 8 * i));
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[hf][8 * i + 2 * e] = bf16_bits_to_float(w[e] & 0xFFFFu);
          x[hf][8 * i + 2 * e + 1] = bf16_bits_to_float(w[e] >> 16);
          amax = fmaxf(amax, fmaxf(fabsf(x[hf][8 * i + 2 * e]), fabsf(x[hf][8 * i + 2 * e + 1])));
        }
      }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    int ex = (int)((__float_as_uint(amax) >> 23) & 0xFF);
    ex = ex < 1 ? 1 : (ex > 253 ? 253 : ex);
    const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
    for (int hf = 0; hf < DH; ++hf)
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const __half2 b0 = __floats2half2_rn(x[hf][4 * w] * down, x[hf][4 * w + 1] * down);
        const __half2 b1 = __floats2half2_rn(x[hf][4 * w + 2] * down, x[hf][4 * w + 3] * down);
        s_qf[(nt * KS + hf * 8 + w) * 32 + lane] = make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
      }
    if (tq == 0) {
      s_mul[col] = up * p.score_scale;
      s_vis[col] = !real || !p.causal ? len : min(len, max(0, hidden + tok));
    }
  }
  __syncthreads();
  int least = len;                        // what every row sees
  for (int c = 0; c < COLS; ++c) least = min(least, s_vis[c]);

  float m[NT][2], l[NT][2], r = 0.f, inv_r = 0.f;
  float o[NT][KS][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int j = 0; j < KS; ++j) { o[t][j][0] = o[t][j][1] = o[t][j][2] = o[t][j][3] = 0.f; }
  }

  for (int i = 0; i < n; ++i) {
    const int s = i % S;
    const bool ok = mbar_wait(my_bar + 8 * s, (i / S) & 1, timed_out, p.status);
    __syncwarp();
    const float2 c = s_sc[warp][s];
    const int tok0 = (u0 + i * kWarps) * kRowsU;
    if (ok && c.x >= 0.f) {
      const uint32_t kt = my_ring + s * P::SLOT, vt = kt + kRowsU * D;
      float sacc[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) { sacc[t][0] = sacc[t][1] = sacc[t][2] = sacc[t][3] = 0.f; }
#pragma unroll
      for (int hf = 0; hf < DH; ++hf)
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          const uint32_t off = hf * (kRowsU * 128) + (((2 * tq + ch) ^ gq) << 4);
          const uint4 klo = lds128(kt + off + gq * 128), khi = lds128(kt + off + (gq + 8) * 128);
          const uint32_t wl[4] = {klo.x, klo.y, klo.z, klo.w}, wh[4] = {khi.x, khi.y, khi.z, khi.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = cvt_lo(wl[w]), a1 = cvt_lo(wh[w]), a2 = cvt_hi(wl[w]), a3 = cvt_hi(wh[w]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const uint2 qf = s_qf[(t * KS + hf * 8 + ch * 4 + w) * 32 + lane];
              mma_f16(sacc[t], a0, a1, a2, a3, qf.x, qf.y);
            }
          }
        }
      float grow = 1.f;
      if (c.y > r) {                      // a page with a larger V scale (the same for the whole warp)
        const float louder = fmaxf(c.y, kLeastScale);
        grow = r / louder;
        r = louder;
        inv_r = 1.f / r;
      }
      const float vs = c.y * inv_r;
      const bool open = tok0 + kRowsU <= least;
      uint32_t pb[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 mul = *reinterpret_cast<const float2*>(s_mul + 8 * t + 2 * tq);
        float s0 = sacc[t][0] * (mul.x * c.x), s1 = sacc[t][1] * (mul.y * c.x), s2 = sacc[t][2] * (mul.x * c.x), s3 = sacc[t][3] * (mul.y * c.x);
        if (!open) {
          const int2 vis = *reinterpret_cast<const int2*>(s_vis + 8 * t + 2 * tq);
          if (tok0 + gq >= vis.x) s0 = -INFINITY;
          if (tok0 + gq >= vis.y) s1 = -INFINITY;
          if (tok0 + gq + 8 >= vis.x) s2 = -INFINITY;
          if (tok0 + gq + 8 >= vis.y) s3 = -INFINITY;
        }
        float mx0 = fmaxf(s0, s2), mx1 = fmaxf(s1, s3);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        const float n0 = fmaxf(m[t][0], mx0), n1 = fmaxf(m[t][1], mx1);
        const float b0 = n0 == -INFINITY ? 0.f : n0 - kPBits, b1 = n1 == -INFINITY ? 0.f : n1 - kPBits;
        float a0 = ex2(m[t][0] - kPBits - b0), a1 = ex2(m[t][1] - kPBits - b1);
        const float p0 = ex2(s0 - b0), p1 = ex2(s1 - b1), p2 = ex2(s2 - b0), p3 = ex2(s3 - b1);
        m[t][0] = n0; m[t][1] = n1;
        l[t][0] = l[t][0] * a0 + (p0 + p2);
        l[t][1] = l[t][1] * a1 + (p1 + p3);
        a0 *= grow; a1 *= grow;
        if (__any_sync(0xffffffffu, a0 != 1.f || a1 != 1.f)) {
#pragma unroll
          for (int j = 0; j < KS; ++j) { o[t][j][0] *= a0; o[t][j][1] *= a1; o[t][j][2] *= a0; o[t][j][3] *= a1; }
        }
        const __half2 pa = __floats2half2_rn(p0 * vs, p1 * vs), pc = __floats2half2_rn(p2 * vs, p3 * vs);
        pb[t][0] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&pa));
        pb[t][1] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&pc));
      }
      const bool tail = tok0 + kRowsU > len;
#pragma unroll
      for (int hf = 0; hf < DH; ++hf) {
        const uint32_t vb = vt + hf * (kRowsU * 128) + 2 * tq * 128;
        uint4 va = lds128(vb + ((gq ^ (2 * tq)) << 4)), vbb = lds128(vb + 128 + ((gq ^ (2 * tq + 1)) << 4));
        uint4 vc = lds128(vb + 1024 + ((gq ^ (2 * tq)) << 4)), vd = lds128(vb + 1152 + ((gq ^ (2 * tq + 1)) << 4));
        if (tail) {                       // slots behind the last token may hold anything, NaN patterns included
          const int tv = tok0 + 2 * tq;
          const uint4 z = make_uint4(0, 0, 0, 0);
          if (tv >= len) va = z;
          if (tv + 1 >= len) vbb = z;
          if (tv + 8 >= len) vc = z;
          if (tv + 9 >= len) vd = z;
        }
        const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vbb.x, vbb.y, vbb.z, vbb.w};
        const uint32_t wc[4] = {vc.x, vc.y, vc.z, vc.w}, wd[4] = {vd.x, vd.y, vd.z, vd.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t x01 = prmt(wa[w], wb[w], 0x5140), x23 = prmt(wa[w], wb[w], 0x7362), y01 = prmt(wc[w], wd[w], 0x5140), y23 = prmt(wc[w], wd[w], 0x7362);
          const uint32_t e0 = cvt_lo(x01), e1 = cvt_hi(x01), e2 = cvt_lo(y01), e3 = cvt_hi(y01);
          const uint32_t f0 = cvt_lo(x23), f1 = cvt_hi(x23), f2 = cvt_lo(y23), f3 = cvt_hi(y23);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16(o[t][hf * 8 + 2 * w], e0, e1, e2, e3, pb[t][0], pb[t][1]);
            mma_f16(o[t][hf * 8 + 2 * w + 1], f0, f1, f2, f3, pb[t][0], pb[t][1]);
          }
        }
      }
    }
    __syncwarp();                         // all lanes have read the slot
    if (!ok) break;
    if (issued < n) issue(issued++);
  }
  if (*timed_out && lane == 0) {
    // A wait ran out.  Copies already issued still land in this block's shared memory: wait for them (bounded).
    for (int s = 0; s < S && s < issued; ++s) {
      const int last = ((issued - 1 - s) / S) * S + s;
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(my_bar + 8 * s, (last / S) & 1) && global_timer_ns() - t0 < kWaitBudgetNs) {}
    }
  }
  __syncthreads();                        // every ring is empty: the states go there

  float* s_acc = reinterpret_cast<float*>(ring_ptr);   // [warp][column][D]
  auto sum_of = [&](float x) { return x * kPUnit * r; };
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[t][hh] += __shfl_xor_sync(0xffffffffu, l[t][hh], off);
      const int col = 8 * t + 2 * tq + hh;
      if (gq == 0) { s_ml[warp][0][col] = m[t][hh]; s_ml[warp][1][col] = l[t][hh] * kPUnit; }
      float* dst = s_acc + (warp * COLS + col) * D + 16 * gq;
#pragma unroll
      for (int hf = 0; hf < DH; ++hf)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<float4*>(dst + hf * 128 + 4 * (w ^ (gq >> 1 & 3))) =
              make_float4(sum_of(o[t][hf * 8 + 2 * w][hh]), sum_of(o[t][hf * 8 + 2 * w][2 + hh]),
                          sum_of(o[t][hf * 8 + 2 * w + 1][hh]), sum_of(o[t][hf * 8 + 2 * w + 1][2 + hh]));
    }
  }
  __syncthreads();
  if (*timed_out) return;
  const long long block = blockIdx.x / p.splits, stride = (long long)COLS * D + 2 * COLS;
  float* part = p.part + block * p.splits * stride;
  const int used = ntok * G * (D / 4);
  auto write = [&](int i, float4 a, float L) {
    const int col = i / (D / 4);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
    reinterpret_cast<uint2*>(p.out + (row0 + (long long)(col / G) * g.h_q + col % G) * D)[i % (D / 4)] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  };
  for (int i = tid; i < used; i += kThreads) {
    const int col = i / (D / 4), d4 = i % (D / 4);
    const int at = (d4 & ~3) | ((d4 & 3) ^ (d4 >> 3 & 3));   // where the lane with these dims has put them
    float M = s_ml[0][0][col];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_ml[w][0][col]);
    float L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_ml[w][0][col] == -INFINITY ? 0.f : ex2(s_ml[w][0][col] - M);
      const float4 v = reinterpret_cast<const float4*>(s_acc + (w * COLS + col) * D)[at];
      L += s_ml[w][1][col] * f;
      a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
    }
    if (pieces == 1) {
      write(i, a, L);
    } else {
      reinterpret_cast<float4*>(part + piece * stride)[i] = a;
      if (d4 == 0) { part[piece * stride + COLS * D + col] = M; part[piece * stride + COLS * D + COLS + col] = L; }
    }
  }
  if (pieces == 1) return;

  // ---- the last piece to be finished joins all of them ----
  __threadfence();
  __syncthreads();
  if (tid == 0) s_info[6] = atomicAdd(p.counters + block, 1) == pieces - 1;
  __syncthreads();
  if (!s_info[6]) return;
  __threadfence();
  if (tid == 0) p.counters[block] = 0;
  for (int i = tid; i < used; i += kThreads) {
    const int col = i / (D / 4);
    float M = -INFINITY, L = 0.f, f[kMostPieces];
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < kMostPieces; ++s) {
      f[s] = s < pieces ? __ldcg(part + s * stride + COLS * D + col) : -INFINITY;
      M = fmaxf(M, f[s]);
    }
#pragma unroll
    for (int s0 = 0; s0 < kMostPieces; s0 += 4) {
      if (s0 >= pieces) break;
      float4 v[4];
      float ls[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float* from = part + min(s0 + s, pieces - 1) * stride;
        v[s] = __ldcg(reinterpret_cast<const float4*>(from) + i);
        ls[s] = __ldcg(from + COLS * D + COLS + col);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float w = f[s0 + s] == -INFINITY ? 0.f : ex2(f[s0 + s] - M);
        L += ls[s] * w;
        a.x += v[s].x * w; a.y += v[s].y * w; a.z += v[s].z * w; a.w += v[s].w * w;
      }
    }
    write(i, a, L);
  }
}

int few_blocks(const PagedGeometry& g) { return g.head_dim == 128 ? FewPlan<128, kTilesN>::BLOCKS : FewPlan<256, kTilesN>::BLOCKS; }

}  // namespace

// The host knows the tokens and sequences of a call, not how they are spread.  A sequence with more rows than a tile takes several,
// each of which reads the keys again; single tokens beside enough others for the larger tiles take 128 rows each.  (Caches of 8192 tokens,
// 40 / 8 heads of 128: 255 single tokens and one chunk of 500 in one call 1184 us, in two calls 723 + 146.)
bool few_rows(const PagedGeometry& g, int n_tokens) {
  return ((long long)n_tokens + g.batch - 1) / g.batch * g.group <= kFewRows && (long long)g.n_pages * g.h_kv * g.page_size <= 0x7fffffffLL;
}

cudaError_t launch_paged_few(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  Geometry cache{};
  cache.n_layers = g.n_layers; cache.batch = g.n_pages; cache.h_kv = g.h_kv; cache.capacity = g.page_size; cache.head_dim = g.head_dim;
  CUtensorMap kmap, vmap;
  if (!encode_cache_map(&kmap, a.k_pages, cache, g.k_layer_stride, kRowsU) || !encode_cache_map(&vmap, a.v_pages, cache, g.v_layer_stride, kRowsU))
    return cudaErrorInvalidValue;
  FewParams p{};
  p.g = g;
  p.q = (const uint16_t*)a.q;
  p.k_scale = a.k_scale; p.v_scale = a.v_scale;
  p.page_table = a.page_table; p.seq_len = a.seq_len; p.q_start = a.q_start;
  p.n_tokens = a.n_tokens;
  p.causal = a.causal;
  p.page_shift = g.page_size == 16 ? 4 : g.page_size == 32 ? 5 : g.page_size == 64 ? 6 : 7;
  p.per_tile = kFewRows / g.group;
  const long long most_tiles = (long long)a.n_tokens / p.per_tile + g.batch;
  p.tiles = (int)(most_tiles < a.n_tokens ? most_tiles : a.n_tokens);
  p.score_scale = a.softmax_scale * kLog2e;
  // As many pieces as the GPU has room for if every sequence makes one tile.  (They cannot make more than twice
  // as many: the average sequence fits in a tile.)
  const long long cap = (long long)g.max_pages * g.page_size, most = a.max_seq_len > 0 && a.max_seq_len < cap ? a.max_seq_len : cap;
  const long long heads = (long long)g.h_kv * g.n_layers, by_len = (most + kLeastUnits * kRowsU - 1) / (kLeastUnits * kRowsU);
  long long splits = (long long)few_blocks(g) * device_sms() / (heads * (g.batch < p.tiles ? g.batch : p.tiles));
  if (splits > by_len) splits = by_len;
  p.splits = (int)(splits < 1 ? 1 : splits > kMostPieces ? kMostPieces : splits);
  p.counters = paged_counters(a.workspace);
  p.part = paged_partials(a.workspace);
  p.out = (uint16_t*)a.out;
  p.status = a.status;
  const long long grid = heads * p.tiles * p.splits;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  auto launch = [&](auto kernel, int smem) -> cudaError_t {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, (int)grid, kThreads, (size_t)smem, stream, kmap, vmap, p);
  };
  return g.head_dim == 128 ? launch(paged_few_kernel<128, kTilesN>, FewPlan<128, kTilesN>::SMEM)
                           : launch(paged_few_kernel<256, kTilesN>, FewPlan<256, kTilesN>::SMEM);
}

size_t paged_few_partial_bytes(const PagedGeometry& g) {
  // split calls have at most twice the blocks that the GPU has room for, counting those that find no tile
  return (size_t)2 * few_blocks(g) * device_sms() * ((size_t)kFewRows * (g.head_dim + 2)) * 4;
}

}  // namespace b200attn
