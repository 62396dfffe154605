// Attention of many query tokens per sequence over the paged FP8 cache, on the 5th-generation tensor cores.
//
//   S = Q K^T * k_scale[page] * softmax_scale * log2(e),  O = sum_t 2^(S_t - m) v_t * v_scale[page] / sum_t 2^(S_t - m)
//
// A thread block owns one tile of 128 query rows of one (layer, sequence, kv head): 128 / G tokens times the G query
// heads that share the kv head, so that a key serves all of them; it walks the visible keys 128 at a time.
//   * K stays in 8 bits: the tile's bytes go from TMA to the tensor core.  A query row is normalised by a power of two and
//     written once as two e4m3 rows, leading part + remainder (a bf16 value has 8 significant bits, e4m3 holds 4): two
//     kind::f8f6f4 products cost what one 16-bit product would, and no key is converted.
//   * V is widened to f16 by four warps on its way from global to shared memory (exact; times the page's scale relative to
//     the largest scale of the block's keys), because P needs more than 8 bits: P is f16 in tensor memory, in the columns
//     that its scores left, and O += P V is kind::f16 with P as the tensor-memory operand.
//   * softmax: one thread per row; scores are read twice from tensor memory (maximum, then exponentials), which keeps the
//     registers few.  The reference maximum moves only when a tile exceeds it by 2^4, so O is rarely rescaled.
//   * heads of 128: two groups of softmax warps take alternate tiles, each with its own maximum, sum and O, joined at the
//     end; heads of 256: one group (O fills the tensor memory, and the products take twice as long per tile).
// Tensor memory: S0 S1 at columns 0 and 128, O at 256 (two of 128 columns, or one of 256).
//
// Bound: the tensor cores (4 D flops per row, key and head), and as much the exponentials, one per row and key:
// 16 a cycle per SM make 1024 cycles a tile, the products of a 128-wide head 1048.
//
// Few rows on a long cache: the keys are cut into pieces over several thread blocks, which leave (m, l, O) in the
// workspace; the last one to finish joins them in order.  Nobody waits for another thread block; waits inside one are bounded.
#include "paged.cuh"
#include "tcgen05.cuh"

namespace b200attn {

namespace {

constexpr int kRows = 128;                 // query rows of a tile
constexpr int kKeys = 128;                 // keys of a tile
constexpr int kInfo = 8;                   // tiles whose scales are in flight
constexpr int kVRing = 3;                  // V units of 32 KB in f16
constexpr int kUnitBytes = 32768;
constexpr float kTauP = 4.f, kBitsP = 11.f;   // p <= 2^4, held times 2^11 in f16
constexpr float kVUp = 128.f;              // V is held times 2^7 (448 * 2^7 < 65504)

struct PrefillParams {
  PagedGeometry g;
  const uint16_t* q;
  const uint8_t* v_pages;
  const float *k_scale, *v_scale;
  const int *page_table, *seq_len, *q_start;
  int n_tokens, causal, page_shift, tiles, splits;     // tiles: upper bound of the query tiles of one layer
  float score_scale;
  float* part;                             // [query tiles * heads * layers][splits][128 * (D + 2)]
  int* counters;
  uint16_t* out;
  int* status;
};

template <int D>
struct PrefillPlan {
  static constexpr int DH = D / 128;
  static constexpr int NS = D == 128 ? 2 : 1;              // softmax groups
  static constexpr int KST = D == 128 ? 3 : 2;             // K tiles in flight
  static constexpr int KTILE = kKeys * D;
  static constexpr int UNIT_KEYS = kUnitBytes / (2 * D);   // keys of a V unit
  static constexpr int UNITS = kKeys / UNIT_KEYS;          // V units of a tile
  static constexpr int WARPS = 4 * NS + 4 + 2;             // softmax, V, TMA, MMA
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SMEM = 1024 + 2 * kRows * D + KST * KTILE + kVRing * kUnitBytes;
};

__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
#define B200_R32(r) \
  "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), \
  "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), \
  "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), \
  "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {   // not complete before tmem_wait32
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : B200_R32(r)::"memory"); }
__device__ __forceinline__ void tmem_st16_nowait(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st32_nowait(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// MN-major operand, 128-byte swizzle: rows (keys) of 128 bytes, 8-row groups 1024 bytes apart, the next 64 f16 dims `lbo` bytes on.
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <int D>
__global__ void __launch_bounds__(PrefillPlan<D>::THREADS, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap kmap, const PrefillParams p) {
  using P = PrefillPlan<D>;
  constexpr int DH = P::DH, NS = P::NS, KST = P::KST;
  constexpr int kSoftmaxWarps = 4 * NS, kFirstV = kSoftmaxWarps, kTma = kSoftmaxWarps + 4, kMma = kSoftmaxWarps + 5;
  // D f32, A and B e4m3, both K-major, N = 128 keys, M = 128;   D f32, A f16 in tensor memory, B f16 MN-major, N = D, M = 128
  constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
  const PagedGeometry& g = p.g;
  const int G = g.group;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  __shared__ __align__(8) uint64_t bars[1 + 2 * KST + kInfo + 2 * kVRing + 6];
  // each 16 keys of a tile: K scale (-1: no such page), V scale, page (-1: none)
  __shared__ __align__(16) float s_ks[kInfo][8], s_vs[kInfo][8];
  __shared__ __align__(16) int s_id[kInfo][8];
  __shared__ float s_red[4];
  __shared__ float s_ml[2][2][kRows];
  __shared__ int s_info[8];                                 // [0] sequence [1] tile of it [2] gave up [3] tensor memory [4] last
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem0, sK = sQ + 2 * kRows * D, sV = sK + KST * P::KTILE;
  const uint32_t qready = smem_u32(bars), kfull = qready + 8, kempty = kfull + 8 * KST, kinfo = kempty + 8 * KST;
  const uint32_t vfull = kinfo + 8 * kInfo, vempty = vfull + 8 * kVRing;
  const uint32_t sfull = vempty + 8 * kVRing, pfull = sfull + 16, odone = pfull + 16;
  volatile int* gave_up = s_info + 2;

  // ---- which tile: piece fastest, then head, layer, query tile from the last (most keys) to the first ----
  const int piece = (int)(blockIdx.x % p.splits);
  int rest = blockIdx.x / p.splits;
  const int h = rest % g.h_kv;
  rest /= g.h_kv;
  const int layer = rest % g.n_layers, number = p.tiles - 1 - rest / g.n_layers;
  const int per_tile = kRows / G;                           // query tokens of a tile
  if (warp == 0) {
    int before = 0;
    if (lane == 0) s_info[0] = -1;
    __syncwarp();
    for (int b0 = 0; b0 < g.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b < g.batch) {
        const int q0 = p.q_start[b], nq = p.q_start[b + 1] - q0;
        if (nq > 0 && q0 >= 0 && q0 + nq <= p.n_tokens) n = (nq + per_tile - 1) / per_tile;
      }
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += t;
      }
      const int start = before + inc - n;
      if (n > 0 && number >= start && number < start + n) { s_info[0] = b; s_info[1] = number - start; }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > number) break;
    }
  }
  if (tid == 32) {
    mbar_init(qready, kSoftmaxWarps);
    for (int i = 0; i < KST; ++i) { mbar_init(kfull + 8 * i, 1); mbar_init(kempty + 8 * i, 1); }
    for (int i = 0; i < kInfo; ++i) mbar_init(kinfo + 8 * i, 1);
    for (int i = 0; i < kVRing; ++i) { mbar_init(vfull + 8 * i, 4); mbar_init(vempty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(sfull + 8 * i, 1); mbar_init(pfull + 8 * i, 4); mbar_init(odone + 8 * i, 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    s_info[2] = 0;
  }
  __syncthreads();
  const int b = s_info[0];
  if (b < 0) return;                                        // the grid is an upper bound
  const int q0 = p.q_start[b], nq = p.q_start[b + 1] - q0;
  const int first_tok = s_info[1] * per_tile, ntok = min(per_tile, nq - first_tok);
  const int len = paged_len(g, p.seq_len[b], p.status, tid == 0 && layer == 0 && h == 0 && piece == 0);
  const int visible = p.causal ? min(len, max(0, len - nq + first_tok + ntok)) : len;   // of the tile's last token
  const int all_tiles = (visible + kKeys - 1) / kKeys;
  const int per_piece = (all_tiles + p.splits - 1) / p.splits;
  const int pieces = per_piece > 0 ? (all_tiles + per_piece - 1) / per_piece : 0;
  const long long out_row0 = ((long long)layer * p.n_tokens + q0 + first_tok) * g.h_q + h * G;   // of (token 0, head 0)
  if (piece >= pieces) {
    if (pieces == 0 && piece == 0)                          // nothing to see: zeros
      for (int i = tid; i < ntok * G * (D / 8); i += P::THREADS) {
        const int row = i / (D / 8);
        reinterpret_cast<uint4*>(p.out + (out_row0 + (long long)(row / G) * g.h_q + row % G) * D)[i % (D / 8)] = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  const int j0 = piece * per_piece, nt = min(per_piece, all_tiles - j0);
  const int key_end = min(len, (j0 + nt) * kKeys);

  if (warp == kMma) tmem_alloc(smem_u32(s_info + 3), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)s_info[3];

  float r_v = 0.f;                                          // largest V scale of the block's keys (V and softmax warps)
  if (warp == kTma) {
    // ================= K tiles; pages and scales of their keys =================
    // Lane i < 8 looks after the tile's keys 16 i .. 16 i + 15.  A page's number and then its scales are two dependent loads, so
    // they run ahead: pages by four tiles, scales by three; they are published two tiles ahead of the K copy (the V warps
    // start from them).  A slot of the ring of kInfo tiles is free by then: K tile j is copied after S(j - KST), i.e. after the
    // softmax of tile j - KST - 2 and the V units of tile j - KST - 2, and j - KST - 2 >= j + 2 - kInfo.
    static_assert(kInfo >= KST + 4, "info ring");
    int issued = 0;
    auto page_at = [&](int j) -> int {
      const int key = (j0 + j) * kKeys + lane * 16;
      return lane < 8 && j < nt && key < key_end ? __ldg(p.page_table + (long long)b * g.max_pages + (key >> p.page_shift)) : -2;   // -2: no key
    };
    auto scales_at = [&](int id) -> float2 {
      if (id == -2) return make_float2(0.f, 0.f);
      if (id < 0 || id >= g.n_pages) return make_float2(-1.f, 0.f);
      const long long si = ((long long)layer * g.n_pages + id) * g.h_kv + h;
      return make_float2(__ldg(p.k_scale + si), __ldg(p.v_scale + si));
    };
    auto publish = [&](int j, int id, float2 sc) {
      if (j >= nt) return;
      if (lane < 8) {
        const bool bad = id != -2 && (id < 0 || id >= g.n_pages);
        if (bad) atomicOr(p.status, B200ATTN_STATUS_BAD_PAGE);
        s_ks[j % kInfo][lane] = sc.x;
        s_vs[j % kInfo][lane] = sc.y;
        s_id[j % kInfo][lane] = bad ? -1 : id;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(kinfo + 8 * (j % kInfo));
    };
    int id0 = page_at(0), id1 = page_at(1), id2 = page_at(2), id3 = page_at(3);
    float2 sc0 = scales_at(id0), sc1 = scales_at(id1), sc2 = scales_at(id2);
    publish(0, id0, sc0);
    publish(1, id1, sc1);
    for (int j = 0; j < nt; ++j) {
      const int st = j % KST;
      const int id4 = page_at(j + 4);
      const float2 sc3 = scales_at(id3);
      if (j >= KST && !mbar_wait_lean(kempty + 8 * st, ((j / KST) - 1) & 1, gave_up, p.status)) break;
      // the lane of a page's first key copies the page
      const bool box = id0 >= 0 && id0 < g.n_pages && ((lane * 16) & (g.page_size - 1)) == 0;
      const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, box));
      if (lane == 0) mbar_arrive_expect_tx(kfull + 8 * st, boxes * g.page_size * D);
      __syncwarp();
      if (box) {
#pragma unroll
        for (int hf = 0; hf < DH; ++hf)
          tma_load_3d(sK + st * P::KTILE + hf * kKeys * 128 + lane * 16 * 128, &kmap, hf * 128, (id0 * g.h_kv + h) << p.page_shift, layer, kfull + 8 * st);
      }
      ++issued;
      publish(j + 2, id2, sc2);
      id0 = id1; id1 = id2; id2 = id3; id3 = id4;
      sc2 = sc3;
    }
    if (lane == 0) s_info[5] = issued;
  } else if (warp == kMma) {
    // ================= products =================
    int s_issued = 0, o_issued = 0;
    bool ok = mbar_wait_lean(qready, 0, gave_up, p.status);
    const uint64_t descQ = smem_desc_k128(sQ), descK = smem_desc_k128(sK);
    const uint64_t descV = smem_desc_mn128(sV, P::UNIT_KEYS * 128);
    auto issue_s = [&](int j) {
      const int st = j % KST;
      if (!mbar_wait_lean(kfull + 8 * st, (j / KST) & 1, gave_up, p.status)) return false;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t d = tmem + (uint32_t)(j & 1) * 128u;
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int hf = 0; hf < DH; ++hf)
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
              umma_f8(d, descQ + (uint64_t)((term * DH + hf) * (kRows * 128 >> 4) + kb * 2), descK + (uint64_t)(st * (P::KTILE >> 4) + hf * (kKeys * 128 >> 4) + kb * 2),
                      kIdescS, (term | hf | kb) ? 1u : 0u);
        umma_commit(sfull + 8 * (j & 1));
        umma_commit(kempty + 8 * st);
      }
      __syncwarp();
      ++s_issued;
      return true;
    };
    ok = ok && issue_s(0);
    if (nt > 1) ok = ok && issue_s(1);
    int vu = 0;
    for (int j = 0; j < nt && ok; ++j) {
      ok = mbar_wait_lean(pfull + 8 * (j & 1), (j >> 1) & 1, gave_up, p.status);
#pragma unroll 1
      for (int u = 0; u < P::UNITS && ok; ++u, ++vu) {
        const int st = vu % kVRing;
        ok = mbar_wait_lean(vfull + 8 * st, (vu / kVRing) & 1, gave_up, p.status);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t d = tmem + 256u + (NS == 2 ? (uint32_t)(j & 1) * 128u : 0u);
          const uint32_t a = tmem + (uint32_t)(j & 1) * 128u + (uint32_t)u * (P::UNIT_KEYS / 2);
#pragma unroll
          for (int kb = 0; kb < P::UNIT_KEYS / 16; ++kb)
            umma_f16_ts(d, a + kb * 8, descV + (uint64_t)(st * (kUnitBytes >> 4) + kb * (2048 >> 4)), kIdescO, (j >= NS || u || kb) ? 1u : 0u);
          umma_commit(vempty + 8 * st);
          if (u == P::UNITS - 1) umma_commit(odone + 8 * (j & 1));
        }
        __syncwarp();
      }
      if (ok) ++o_issued;
      if (ok && j + 2 < nt) ok = issue_s(j + 2);
    }
    if (lane == 0) { s_info[6] = s_issued; s_info[7] = o_issued; }
  } else if (warp >= kFirstV) {
    // ================= V: widened to f16 between global and shared memory =================
    const int vw = warp - kFirstV, vt = tid - kFirstV * 32;
    // the largest V scale of the block's keys
    {
      float r = 0.f;
      const int pg0 = j0 * kKeys / g.page_size, pg1 = (key_end - 1) / g.page_size;
      for (int i = pg0 + vt; i <= pg1; i += 128) {
        const int id = p.page_table[(long long)b * g.max_pages + i];
        if (id >= 0 && id < g.n_pages) r = fmaxf(r, p.v_scale[((long long)layer * g.n_pages + id) * g.h_kv + h]);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, off));
      if (lane == 0) s_red[vw] = r;
      asm volatile("bar.sync 2, 128;" ::: "memory");
      r_v = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    }
    const float inv_r = r_v > 0.f ? kVUp / r_v : 0.f;
    const uint8_t* vbase = p.v_pages + (long long)layer * g.v_layer_stride;
    // a lane's 16 bytes: chunk k of 64-dim block blk of row ro; the mapping makes 8 lanes hit all banks when they store
    const int k4 = lane & 3, blk = D == 128 ? (lane >> 3) & 1 : lane >> 3;
    const int ro = ((lane >> 2) & 1) + (D == 128 ? (lane >> 4) * 2 : 0) + vw * (D == 128 ? 4 : 2);
    constexpr int STEP = D == 128 ? 16 : 8;                 // rows of one load of the four warps
    constexpr int N = P::UNIT_KEYS / STEP;                  // loads per lane and unit: 8
    const int units = nt * P::UNITS;
    uint4 raw[2][N];
    auto load = [&](int u, uint4 (&rw)[N]) {
      const int key0 = j0 * kKeys + u * P::UNIT_KEYS + ro, c0 = (u % P::UNITS) * (P::UNIT_KEYS / 16);
      const int* ids = s_id[(u / P::UNITS) % kInfo];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = key0 + i * STEP, id = ids[c0 + i * STEP / 16];
        rw[i] = make_uint4(0, 0, 0, 0);
        if (key < key_end && id >= 0)
          rw[i] = __ldg(reinterpret_cast<const uint4*>(vbase + (((((long long)id * g.h_kv + h) << p.page_shift) + (key & (g.page_size - 1))) * D + blk * 64 + k4 * 16)));
      }
    };
    auto store = [&](int u, int st, const uint4 (&rw)[N]) {
      const uint32_t base = sV + st * kUnitBytes + blk * (P::UNIT_KEYS * 128);
      const float* vs = s_vs[(u / P::UNITS) % kInfo] + (u % P::UNITS) * (P::UNIT_KEYS / 16);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = ro + i * STEP;
        // the page's scale relative to the largest, as leading part + remainder
        const float ratio = vs[i * STEP / 16] * inv_r;
        const __half2 hi = __float2half2_rn(ratio), lo = __float2half2_rn(ratio - __low2float(hi));
        const uint32_t w[4] = {rw[i].x, rw[i].y, rw[i].z, rw[i].w};
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t h2 = e4m3x2_to_f16x2((uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu));
          const __half2 x = *reinterpret_cast<const __half2*>(&h2);
          const __half2 y = __hfma2(x, hi, __hmul2(x, lo));
          o[e] = *reinterpret_cast<const uint32_t*>(&y);
        }
        const uint32_t rowaddr = base + row * 128;
        sts128(rowaddr + (((2 * k4) ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
        sts128(rowaddr + (((2 * k4 + 1) ^ (row & 7)) << 4), o[4], o[5], o[6], o[7]);
      }
    };
    bool alive = mbar_wait_lean(kinfo, 0, gave_up, p.status);
    if (alive) load(0, raw[0]);
#pragma unroll 1
    for (int u = 0; u < units && alive; u += 2) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int uu = u + half;
        if (uu < units && alive) {
          if (uu + 1 < units) {
            const int t = (uu + 1) / P::UNITS;
            if ((uu + 1) % P::UNITS == 0) alive = mbar_wait_lean(kinfo + 8 * (t % kInfo), (t / kInfo) & 1, gave_up, p.status);
            if (alive) load(uu + 1, raw[half ^ 1]);
          }
          const int st = uu % kVRing;
          if (alive && uu >= kVRing) alive = mbar_wait_lean(vempty + 8 * st, ((uu / kVRing) - 1) & 1, gave_up, p.status);
          if (alive) {
            store(uu, st, raw[half]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(vfull + 8 * st);
          }
        }
      }
    }
  } else {
    // ================= softmax: one thread per query row =================
    const int grp = warp >> 2, row = tid & 127;
    const int tok = row / G, head = row % G;
    const bool real = tok < ntok;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint16_t* qrow = p.q + (out_row0 + (long long)tok * g.h_q + head) * D;
    // the query row as two e4m3 rows; with two groups each writes half of the row's dims
    float rowmul;
    {
      float amax = 0.f;
      if (real)
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const uint4 w4 = __ldg(reinterpret_cast<const uint4*>(qrow) + i);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xFFFF0000u))));
        }
      int ex = (int)((__float_as_uint(amax) >> 23) & 0xFF);
      ex = ex < 8 ? 8 : (ex > 253 ? 253 : ex);
      const float down = __uint_as_float((uint32_t)(261 - ex) << 23), up = __uint_as_float((uint32_t)(ex - 7) << 23);   // largest |q| in [128, 256)
      rowmul = up * p.score_scale;
#pragma unroll 2
      for (int c = grp * (D / 16 / NS); c < (grp + 1) * (D / 16 / NS); ++c) {   // 16 dims
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 w4 = make_uint4(0, 0, 0, 0);
          if (real) w4 = __ldg(reinterpret_cast<const uint4*>(qrow) + 2 * c + i);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x0 = __uint_as_float(w[2 * e] << 16) * down, x1 = __uint_as_float(w[2 * e] & 0xFFFF0000u) * down;
            const float x2 = __uint_as_float(w[2 * e + 1] << 16) * down, x3 = __uint_as_float(w[2 * e + 1] & 0xFFFF0000u) * down;
            const float h0 = e4m3_head(x0), h1 = e4m3_head(x1), h2 = e4m3_head(x2), h3 = e4m3_head(x3);
            hi[2 * i + e] = pack_e4m3x2(h0, h1) | (pack_e4m3x2(h2, h3) << 16);
            lo[2 * i + e] = pack_e4m3x2(x0 - h0, x1 - h1) | (pack_e4m3x2(x2 - h2, x3 - h3) << 16);
          }
        }
        const uint32_t off = (uint32_t)(c >> 3) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        sts128(sQ + off, hi[0], hi[1], hi[2], hi[3]);
        sts128(sQ + DH * kRows * 128 + off, lo[0], lo[1], lo[2], lo[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(qready);
    }
    // keys this row sees; rows of no token see all of them (their results go nowhere, and they need no mask)
    const int vis = !real ? 0x7fffffff : p.causal ? min(len, max(0, len - nq + first_tok + tok + 1)) : len;

    float m = -INFINITY, l = 0.f;
    bool alive = true;
    for (int j = grp; j < nt && alive; j += NS) {
      const int base = (j0 + j) * kKeys;
      alive = mbar_wait_lean(kinfo + 8 * (j % kInfo), (j / kInfo) & 1, gave_up, p.status);
      if (alive) alive = mbar_wait_lean(sfull + 8 * (j & 1), (j >> 1) & 1, gave_up, p.status);
      if (!alive) break;
      tc_fence_after();
      float a[8];
      bool bad = false;
      {
        const float4 x = *reinterpret_cast<const float4*>(s_ks[j % kInfo]), y = *reinterpret_cast<const float4*>(s_ks[j % kInfo] + 4);
        a[0] = x.x; a[1] = x.y; a[2] = x.z; a[3] = x.w; a[4] = y.x; a[5] = y.y; a[6] = y.z; a[7] = y.w;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          bad |= a[c] < 0.f;
        }
      }
      const bool mask = !__all_sync(0xffffffffu, vis >= base + kKeys) || bad;
      const uint32_t ts = tmem + lane_base + (uint32_t)(j & 1) * 128u;
      // ---- maximum: the next 32 scores are on their way while these are looked at ----
      float tmax = -INFINITY;
      uint32_t s[2][32];
      tmem_ld32(ts, s[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t (&x)[32] = s[c & 1];
        tmem_wait32(x);
        tmem_ld32(ts + 32 * ((c + 1) & 3), s[(c + 1) & 1]);   // after the last: the first again, for the exponentials
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float mx = -INFINITY;
          if (!mask) {
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, __uint_as_float(x[16 * hh + i]));
          } else {
            const int n = a[2 * c + hh] < 0.f ? 0 : vis - base - 32 * c - 16 * hh;   // keys of these 16 that the row sees
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, i < n ? __uint_as_float(x[16 * hh + i]) : -INFINITY);
          }
          tmax = fmaxf(tmax, mx == -INFINITY ? -INFINITY : mx * (rowmul * a[2 * c + hh]));
        }
      }
      // ---- the reference moves when a tile exceeds it by more than kTauP ----
      float alpha = 1.f;
      if (tmax > m + kTauP || m == -INFINITY) {
        alpha = m == -INFINITY ? 0.f : ex2(m - tmax);
        m = tmax;
        l *= alpha;
      }
      if (j >= NS && __any_sync(0xffffffffu, alpha != 1.f)) {
        if (NS == 1) {                                      // the product of the tile before (two groups: complete, since these scores are)
          alive = mbar_wait_lean(odone + 8 * ((j - 1) & 1), ((j - 1) >> 1) & 1, gave_up, p.status);
          if (!alive) break;
          tc_fence_after();
        }
        const uint32_t to = tmem + lane_base + 256u + (uint32_t)grp * 128u;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          tmem_ld32(to + 32 * c, s[1]);
          tmem_wait32(s[1]);
#pragma unroll
          for (int i = 0; i < 32; ++i) s[1][i] = __float_as_uint(__uint_as_float(s[1][i]) * alpha);
          tmem_st32_nowait(to + 32 * c, s[1]);
        }
      }
      // ---- probabilities, into the columns that the scores leave ----
      const float mb = (m == -INFINITY ? 0.f : m) - kBitsP;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t (&x)[32] = s[c & 1];
        tmem_wait32(x);
        if (c < 3) tmem_ld32(ts + 32 * (c + 1), s[(c + 1) & 1]);
        uint32_t pk[16];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float f = rowmul * a[2 * c + hh];
          const int n = !mask ? 16 : a[2 * c + hh] < 0.f ? 0 : vis - base - 32 * c - 16 * hh;
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float p0 = ex2(fmaf(__uint_as_float(x[16 * hh + i]), f, -mb)), p1 = ex2(fmaf(__uint_as_float(x[16 * hh + i + 1]), f, -mb));
            if (mask) {
              p0 = i < n ? p0 : 0.f;
              p1 = i + 1 < n ? p1 : 0.f;
            }
            sum0 += p0;
            sum1 += p1;
            const __half2 h2 = __floats2half2_rn(p0, p1);
            pk[8 * hh + i / 2] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          l += sum0 + sum1;
        }
        tmem_st16_nowait(ts + 16 * c, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull + 8 * (j & 1));
    }

    // ---- the end: this group's last product ----
    const int mine = (nt - grp + NS - 1) / NS;              // tiles of this group
    if (alive && mine > 0) {
      const int jl = grp + (mine - 1) * NS;
      alive = mbar_wait_lean(odone + 8 * (jl & 1), (jl >> 1) & 1, gave_up, p.status);
      tc_fence_after();
    }
    if (NS == 2) {
      s_ml[grp][0][row] = m;
      s_ml[grp][1][row] = l;
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");
      tc_fence_after();
    }
    r_v = s_red[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) r_v = fmaxf(r_v, s_red[i]); // written before the first V unit was
    float f0 = 1.f, f1 = 0.f, M = m, L = l;
    if (NS == 2) {
      const float m0 = s_ml[0][0][row], m1 = s_ml[1][0][row];
      M = fmaxf(m0, m1);
      f0 = m0 == -INFINITY ? 0.f : ex2(m0 - M);
      f1 = m1 == -INFINITY ? 0.f : ex2(m1 - M);
      L = s_ml[0][1][row] * f0 + s_ml[1][1][row] * f1;
    }
    const float unit = r_v * (1.f / kVUp);
    const float scale = pieces > 1 ? unit : (L > 0.f ? unit / L : 0.f);
    float* part = p.part + ((long long)(blockIdx.x / p.splits) * p.splits + piece) * (kRows * (D + 2));
    if (alive && !*gave_up) {
#pragma unroll 1
      for (int c = grp * (D / 32 / NS); c < (grp + 1) * (D / 32 / NS); ++c) {
        uint32_t x[32];
        float o[32];
        tmem_ld32(tmem + lane_base + 256u + 32 * c, x);
        tmem_wait32(x);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = f0 == 0.f ? 0.f : __uint_as_float(x[i]) * f0;
        if (NS == 2 && nt > 1) {
          tmem_ld32(tmem + lane_base + 384u + 32 * c, x);
          tmem_wait32(x);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] += f1 == 0.f ? 0.f : __uint_as_float(x[i]) * f1;
        }
        if (real && pieces == 1) {
          uint4* dst = reinterpret_cast<uint4*>(p.out + (out_row0 + (long long)tok * g.h_q + head) * D + 32 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 v2 = __floats2bfloat162_rn(o[8 * i + 2 * e] * scale, o[8 * i + 2 * e + 1] * scale);
              w[e] = *reinterpret_cast<const uint32_t*>(&v2);
            }
            dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (real) {
          float4* dst = reinterpret_cast<float4*>(part + (long long)row * D + 32 * c);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i] * scale, o[4 * i + 1] * scale, o[4 * i + 2] * scale, o[4 * i + 3] * scale);
        }
      }
      if (pieces > 1 && real && grp == 0) {
        part[kRows * D + row] = M;
        part[kRows * D + kRows + row] = L;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    if (*gave_up && lane == 0) {
      // A wait ran out: wait (bounded) for what was issued into this block's shared and tensor memory.
      auto drain = [&](uint32_t bar, int ring, int issued) {
        for (int s = 0; s < ring && s < issued; ++s) {
          const int last = ((issued - 1 - s) / ring) * ring + s;
          const unsigned long long t0 = global_timer_ns();
          while (!mbar_try_wait(bar + 8 * s, (last / ring) & 1) && global_timer_ns() - t0 < kWaitBudgetNs) {}
        }
      };
      drain(kfull, KST, s_info[5]);
      drain(sfull, 2, s_info[6]);
      drain(odone, 2, s_info[7]);
    }
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (pieces == 1) return;

  // ---- the last piece to be finished joins all of them ----
  const long long tile_id = blockIdx.x / p.splits;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_info[4] = atomicAdd(p.counters + tile_id, 1) == pieces - 1;
  __syncthreads();
  if (!s_info[4]) return;
  __threadfence();
  if (tid == 0) p.counters[tile_id] = 0;
  const float* part = p.part + tile_id * p.splits * (kRows * (D + 2));
  constexpr long long stride = kRows * (D + 2);
  for (int i = tid; i < ntok * G * (D / 4); i += P::THREADS) {
    const int row = i / (D / 4);
    float M = -INFINITY, L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < pieces; ++s) M = fmaxf(M, __ldcg(part + s * stride + kRows * D + row));
#pragma unroll 4
    for (int s = 0; s < pieces; ++s) {
      const float ms = __ldcg(part + s * stride + kRows * D + row);
      const float f = ms == -INFINITY ? 0.f : ex2(ms - M);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(part + s * stride) + i);
      L += __ldcg(part + s * stride + kRows * D + kRows + row) * f;
      a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
    reinterpret_cast<uint2*>(p.out + (out_row0 + (long long)(row / G) * g.h_q + row % G) * D)[i % (D / 4)] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// Query tiles of a layer and head, at most: every sequence can have one that is not full, and has none without tokens.
long long prefill_tiles(const PagedGeometry& g, int n_tokens) {
  const int per_tile = kRows / g.group;
  const long long most = (long long)n_tokens / per_tile + g.batch;
  return most < n_tokens ? most : n_tokens;
}
// Pieces of the keys: where the query tiles do not fill the GPU, as many as do, none under 4 tiles of keys.
int prefill_splits(const PagedGeometry& g, int n_tokens, int max_seq_len) {
  const long long cap = (long long)g.max_pages * g.page_size;
  const long long most = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  const long long blocks = prefill_tiles(g, n_tokens) * g.h_kv * g.n_layers;
  if (blocks < 1) return 1;
  long long want = device_sms() / blocks;
  const long long by_len = (most + 4 * kKeys - 1) / (4 * kKeys);
  if (want > by_len) want = by_len;
  return (int)(want < 1 ? 1 : want);
}

}  // namespace

size_t paged_prefill_workspace_bytes(const PagedGeometry& g, int n_tokens, int max_seq_len) {
  // A workspace serves every call with up to n_tokens query rows; fewer tokens can mean more pieces: tiles * pieces is at
  // most the SM count whenever there are pieces, so that many slots do for all of them.
  (void)n_tokens;
  (void)max_seq_len;
  return (size_t)device_sms() * ((size_t)kRows * (g.head_dim + 2) * 4 + 4) + 16;
}

cudaError_t launch_paged_prefill(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  Geometry cache{};
  cache.n_layers = g.n_layers; cache.batch = g.n_pages; cache.h_kv = g.h_kv; cache.capacity = g.page_size; cache.head_dim = g.head_dim;
  CUtensorMap kmap;
  if (!encode_cache_map(&kmap, a.k_pages, cache, g.k_layer_stride, g.page_size)) return cudaErrorInvalidValue;
  PrefillParams p{};
  p.g = g;
  p.q = (const uint16_t*)a.q;
  p.v_pages = (const uint8_t*)a.v_pages;
  p.k_scale = a.k_scale; p.v_scale = a.v_scale;
  p.page_table = a.page_table; p.seq_len = a.seq_len; p.q_start = a.q_start;
  p.n_tokens = a.n_tokens;
  p.causal = a.causal;
  p.page_shift = g.page_size == 16 ? 4 : g.page_size == 32 ? 5 : g.page_size == 64 ? 6 : 7;
  p.tiles = (int)prefill_tiles(g, a.n_tokens);
  p.splits = prefill_splits(g, a.n_tokens, a.max_seq_len);
  p.score_scale = a.softmax_scale * kLog2e;
  p.counters = (int*)a.workspace;
  p.part = (float*)((uint8_t*)a.workspace + (((size_t)device_sms() * 4 + 15) & ~(size_t)15));
  p.out = (uint16_t*)a.out;
  p.status = a.status;
  const long long grid = (long long)p.tiles * p.splits * g.h_kv * g.n_layers;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  auto launch = [&](auto kernel, int threads, int smem) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)grid, threads, smem, stream>>>(kmap, p);
    return cudaGetLastError();
  };
  return g.head_dim == 128 ? launch(paged_prefill_kernel<128>, PrefillPlan<128>::THREADS, PrefillPlan<128>::SMEM)
                           : launch(paged_prefill_kernel<256>, PrefillPlan<256>::THREADS, PrefillPlan<256>::SMEM);
}

}  // namespace b200attn
