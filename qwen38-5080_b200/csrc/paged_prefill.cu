// Attention of many query tokens per sequence over the paged FP8 cache, on the 5th-generation tensor cores.
//
//   S = Q K^T * k_scale[page] * softmax_scale * log2(e),  O = sum_t 2^(S_t - m) v_t * v_scale[page] / sum_t 2^(S_t - m)
//
// A thread block owns one tile of 128 query rows of one (layer, sequence, kv head): 128 / G tokens times the G query
// heads that share the kv head, so that a key serves all of them; it walks the visible keys 128 at a time.
//   * K stays in 8 bits: the tile's bytes go from TMA to the tensor core.  A query row is normalised by a power of two and
//     written once as two e4m3 rows, leading part + remainder (a bf16 value has 8 significant bits, e4m3 holds 4; exact for
//     elements within 2^9 of the row's largest, smaller ones are off by at most 2^-16 of it): two
//     kind::f8f6f4 products cost what one 16-bit product would, and no key is converted.
//   * V's bytes come by TMA too; four warps widen them to f16, shared memory to shared memory (exact; times the page's scale relative to
//     the largest scale of the block's keys), because P needs more than 8 bits: P is f16 in tensor memory, in the columns
//     that its scores left, and O += P V is kind::f16 with P as the tensor-memory operand.
//   * softmax: one thread per row, which takes 64 scores at a time into registers (the other warps give theirs up for it).  The
//     exponentials are taken against the reference maximum as it stands, without looking for the tile's maximum first; a
//     p far beyond it shows in the sum, and only then the reference moves and O is rescaled.  f16 holds 2^12 above the
//     reference and 2^28 below it, sums and O are fp32: nothing is lost by a reference that is not the maximum.
//   * P is handed over 64 keys at a time, so that they are multiplied while the next exponentials are taken; with heads of 128
//     each 64 keys' scores have a buffer of their own, refilled as soon as their P is multiplied.
//   * heads of 128: two groups of softmax warps, each with its own S, P and O.  With rows enough a block takes two query tiles,
//     one for each group, which share the K copies and the V conversion; otherwise the groups take alternate key tiles of
//     one query tile, joined at the end.  Heads of 256: one group (O fills the tensor memory, and the products take twice as
//     long per tile).
// Tensor memory: S at columns 0..255 (two of 128, or four of 64), O at 256 (one of 256 columns, or two of 128).
//
// Bound: the tensor cores (4 D flops per row, key and head), and as much the exponentials, one per row and key:
// 16 a cycle per SM make 1024 cycles a tile, the products of a 128-wide head 1048; a tile takes 1,800 to 2,100 (heads of 256: 3,400
// for 2,096), a block's start 7,000 (15,000) and its end 4,000.  An 8192-token prompt, 40 / 8 heads of 128: 705 to 730 us by GPU, 0.94 to 0.97 PFLOP/s.
//
// Few rows on a long cache: the keys are cut into pieces over several thread blocks, which leave (m, l, O) in the
// workspace, and a second kernel joins them in order.  Nobody waits for another thread block; waits inside one are bounded.
#include <type_traits>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace b200attn {

namespace {

constexpr int kRows = 128;                 // query rows of a tile
constexpr int kKeys = 128;                 // keys of a tile
constexpr int kInfo = 8;                   // tiles whose scales are in flight
constexpr int kVRing = 2;                  // V units of 32 KB in f16
constexpr int kUnitBytes = 32768;
constexpr float kBitsP = 4.f, kMostP = 61440.f;   // p is held times 2^4 in f16; what 64 keys may add up to before the reference moves
constexpr float kPUnit = 1.f / 16.f;       // pieces are left without that factor: times a loud V scale it could pass the largest float
constexpr int kPolyEvery = 4;              // of every 4 * kPolyEvery exponentials, two by polynomial
constexpr float kVUp = 128.f;              // V is held times 2^7 (448 * 2^7 < 65504)
// V is held relative to the largest scale of the block's keys, but to no less than this: kVUp / 2^-126, which zero values have, is not finite.
// 2^-126 then stands as 2^-8, times 2^7 still exact in f16 for every byte; smaller scales keep what subnormal bf16 outputs can hold.
constexpr float kLeastV = 0x1p-118f;

struct PrefillTile {
  long long row0;                          // output row of (token 0, head 0)
  int rows, pieces;
};
struct PrefillParams {
  PagedGeometry g;
  const uint16_t* q;
  const float *k_scale, *v_scale;
  const int *page_table, *seq_len, *q_start;
  int n_tokens, causal, page_shift, pair, tiles, splits;   // pair: a block takes two query tiles; tiles: upper bound of the query tiles of one layer
  float score_scale;
  float* part;                             // [query tiles * heads * layers][splits][128 * (D + 2)]
  PrefillTile* done;                       // [query tiles * heads * layers], where there are pieces: what to join
  uint16_t* out;
  int* status;
};

template <int D>
struct PrefillPlan {
  static constexpr int DH = D / 128;
  static constexpr int NS = D == 128 ? 2 : 1;              // softmax groups
  static constexpr int KST = D == 128 ? 3 : 2;             // K tiles in flight
  static constexpr int KTILE = kKeys * D;
  static constexpr int SK = D == 128 ? 64 : 128;           // keys of a score buffer; every group has two buffers
  static constexpr int UNIT_KEYS = kUnitBytes / (2 * D);   // keys of a V unit
  static constexpr int UNITS = kKeys / UNIT_KEYS;          // V units of a tile
  static constexpr int RAW = 2;                            // V units in flight as bytes
  static constexpr int QTILE = 2 * kRows * D;              // a query tile as two e4m3 terms
  static constexpr int RAW_BYTES = kUnitBytes / 2;
  static constexpr int WARPS = 4 * NS + 8;                 // softmax, V, and a group of TMA, MMA and two idle warps
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SMEM = 1024 + NS * QTILE + KST * KTILE + kVRing * kUnitBytes + RAW * RAW_BYTES;
  // Registers per thread after the roles part: softmax keeps 64 scores of a row and their P.  The shares add up to what the block
  // is launched with (512 x 128; 384 x 168): 256 x 184 + 256 x 72; 128 x 232 + 256 x 136.
  static constexpr int REGS_SOFTMAX = D == 128 ? 184 : 232;
  static constexpr int REGS_OTHER = D == 128 ? 72 : 136;
};
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// One lane of the warp, as the compiler knows it: what it issues stays in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// Shared-memory operand descriptor from its low word: address / 16, and the leading offset / 16 in the upper half.  8-row groups
// 1024 bytes apart, 128-byte swizzle, sm_100 descriptor version 1 (smem_desc_k128 with the words apart).
__device__ __forceinline__ uint64_t desc_of(uint32_t low) {
  return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | low;
}
__device__ __forceinline__ void umma_s(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {   // e4m3 x e4m3
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d), "l"(desc_of(a)), "l"(desc_of(b)), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
__device__ __forceinline__ void umma_o(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {   // f16 (tensor memory) x f16
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d), "r"(a), "l"(desc_of(b)), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
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
// 64 scores of a row (the load and the wait for it in one statement: the registers are not touched before it is over).
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32_nowait(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// 32 bytes, one full sector, in one store.
__device__ __forceinline__ void stg256(void* dst, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// try_wait that may suspend the warp for up to a millisecond: a waiting warp that polls takes issue slots from the others.
__device__ __forceinline__ bool try_wait_long(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
      : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000000u) : "memory");
  return ok != 0;
}
// Bounded wait without a call: functions that are called would have to fit the registers of the warps that gave theirs up.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
#pragma unroll 1
  while (!try_wait_long(bar, parity)) {
    if (*gave_up) return false;
    if (global_timer_ns() - t0 > kWaitBudgetNs) {
      *gave_up = 1;
      atomicOr(status, B200ATTN_STATUS_WAIT_TIMEOUT);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void tmem_st16_nowait(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// x within [-126, 127]; NaN stays NaN.
__device__ __forceinline__ float within_exponents(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(-126.f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(127.f));
  return r;
}
// 2^x of two values without the special-function unit: x = n + f, n the nearest integer (from the low bits of x + 1.5 2^23), 2^f by
// the degree-3 polynomial of least relative error on [-1/2, 1/2] (Remez exchange; 7.5e-5 = 2^-13.7, against the f16 rounding of
// up to 2^-11 that follows), n added to its exponent.  Above 127 it gives about 2^127, and so does NaN (0x7FFFFFFF << 23 plus 0x7FFFFFFF
// wraps to the largest float): both are far above what the caller accepts of a sum.
__device__ __forceinline__ void ex2_pair(float& x, float& y) {
  const unsigned long long v = pair2(within_exponents(x), within_exponents(y));
  const unsigned long long t = add2(v, pair2(12582912.f, 12582912.f));
  const unsigned long long f = add2(v, fma2(t, pair2(-1.f, -1.f), pair2(12582912.f, 12582912.f)));
  unsigned long long q = fma2(f, pair2(0.0551716691f, 0.0551716691f), pair2(0.242611122f, 0.242611122f));
  q = fma2(q, f, pair2(0.693260985f, 0.693260985f));
  q = fma2(q, f, pair2(0.999928074f, 0.999928074f));
  float t0, t1, q0, q1;
  split2(t, t0, t1);
  split2(q, q0, q1);
  x = __uint_as_float((__float_as_uint(t0) << 23) + __float_as_uint(q0));
  y = __uint_as_float((__float_as_uint(t1) << 23) + __float_as_uint(q1));
}

template <int D>
__global__ void __launch_bounds__(PrefillPlan<D>::THREADS, 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PrefillParams p) {
  using P = PrefillPlan<D>;
  constexpr int DH = P::DH, NS = P::NS, KST = P::KST;
  constexpr int kSoftmaxWarps = 4 * NS, kFirstV = kSoftmaxWarps, kTma = kSoftmaxWarps + 4, kMma = kSoftmaxWarps + 5;
  // D f32, A and B e4m3, both K-major, N = 128 keys, M = 128;   D f32, A f16 in tensor memory, B f16 MN-major, N = D, M = 128
  constexpr uint32_t kIdescS = (1u << 4) | (((uint32_t)P::SK >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
  const PagedGeometry& g = p.g;
  const int G = g.group;
  const int tid = threadIdx.x, lane = tid & 31;
  // Through a shuffle, so that the compiler knows that it is the same in all lanes: roles branch without divergence, and what
  // they compute for all lanes (loop counters, descriptors) stays in uniform registers.
  auto uniform = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
  const int warp = uniform(tid >> 5);

  __shared__ __align__(8) uint64_t bars[1 + 2 * KST + kInfo + 2 * kVRing + 2 * P::RAW + 2 * NS + 8];
  // each 16 keys of a tile: K scale (-1: no such page), V scale, page (-1: none)
  __shared__ __align__(16) float s_ks[kInfo][8], s_vs[kInfo][8];
  __shared__ __align__(16) int s_id[kInfo][8];
  __shared__ float s_red[4];
  __shared__ float s_ml[2][2][kRows], s_rowmul[NS][kRows];
  __shared__ int s_info[10];   // [0] sequence [1] tile of it [2] gave up [3] tensor memory [4] last [5] first row [6] rows [7] length [8] K tiles, [9] V units issued
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem0, sK = sQ + NS * P::QTILE, sV = sK + KST * P::KTILE, sRaw = sV + kVRing * kUnitBytes;
  const uint32_t qready = smem_u32(bars), kfull = qready + 8, kempty = kfull + 8 * KST, kinfo = kempty + 8 * KST;
  const uint32_t vfull = kinfo + 8 * kInfo, vempty = vfull + 8 * kVRing;
  const uint32_t sfull = vempty + 8 * kVRing, pfull = sfull + 16 * NS, odone = pfull + 32;   // of both halves of both buffers
  const uint32_t rfull = odone + 32, rempty = rfull + 8 * P::RAW;
  volatile int* gave_up = s_info + 2;

  // ---- which tile: piece fastest, then head, layer, query tile from the last (most keys) to the first ----
  const int piece = (int)(blockIdx.x % p.splits);
  int rest = blockIdx.x / p.splits;
  const int h = rest % g.h_kv;
  rest /= g.h_kv;
  const int layer = rest % g.n_layers, number = p.tiles - 1 - rest / g.n_layers;
  const int per_tile = kRows / G, per_block = per_tile << p.pair;   // query tokens of a tile, of a block
  pdl_wait();
  if (warp == 0) {
    int before = 0;
    if (lane == 0) s_info[0] = -1;
    __syncwarp();
    for (int b0 = 0; b0 < g.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0, q0 = 0, nq = 0, raw_len = 0;
      if (b < g.batch) {
        q0 = p.q_start[b];
        const int end = p.q_start[b + 1];
        nq = end - q0;
        raw_len = p.seq_len[b];
        if (range_fits(q0, end, p.n_tokens, p.status, blockIdx.x == 0) && nq > 0) n = (nq + per_block - 1) / per_block;
      }
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += t;
      }
      const int start = before + inc - n;
      if (n > 0 && number >= start && number < start + n) { s_info[0] = b; s_info[1] = number - start; s_info[5] = q0; s_info[6] = nq; s_info[7] = raw_len; }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > number && blockIdx.x != 0) break;         // the first block has looked at every sequence
    }
  }
  if (tid == 32) {
    mbar_init(qready, kSoftmaxWarps + (NS == 1 ? 4 : 0));
    for (int i = 0; i < KST; ++i) { mbar_init(kfull + 8 * i, 1); mbar_init(kempty + 8 * i, 1); }
    for (int i = 0; i < kInfo; ++i) mbar_init(kinfo + 8 * i, 1);
    for (int i = 0; i < kVRing; ++i) { mbar_init(vfull + 8 * i, 4); mbar_init(vempty + 8 * i, 1); }
    for (int i = 0; i < P::RAW; ++i) { mbar_init(rfull + 8 * i, 1); mbar_init(rempty + 8 * i, 4); }
    for (int i = 0; i < 2 * NS; ++i) mbar_init(sfull + 8 * i, 1);
    for (int i = 0; i < 4; ++i) { mbar_init(pfull + 8 * i, 4); mbar_init(odone + 8 * i, 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    s_info[2] = 0;
  }
  __syncthreads();
  const int b = uniform(s_info[0]);
  pdl_launch_dependents();
  const bool reports = p.splits > 1 && piece == 0 && tid == 0;
  if (b < 0) {                                              // the grid is an upper bound
    if (reports) p.done[blockIdx.x / p.splits] = PrefillTile{0, 0, 0};
    return;
  }
  const int q0 = uniform(s_info[5]), nq = uniform(s_info[6]);
  const int first_tok = uniform(s_info[1]) * per_block, ntok = min(per_block, nq - first_tok);
  const bool two = NS == 2 && ntok > per_tile;              // two query tiles, one for each softmax group; else they share one
  const int len = paged_len(g, uniform(s_info[7]), p.status, tid == 0 && layer == 0 && h == 0 && piece == 0);
  const int visible = p.causal ? min(len, max(0, len - nq + first_tok + ntok)) : len;   // of the tile's last token
  const int all_tiles = (visible + kKeys - 1) / kKeys;
  const int per_piece = (all_tiles + p.splits - 1) / p.splits;
  const int pieces = per_piece > 0 ? (all_tiles + per_piece - 1) / per_piece : 0;
  const long long out_row0 = ((long long)layer * p.n_tokens + q0 + first_tok) * g.h_q + h * G;   // of (token 0, head 0)
  if (reports) p.done[blockIdx.x / p.splits] = PrefillTile{out_row0, ntok * G, pieces};
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

  B200ATTN_CHECK(p.status, first_tok >= 0 && ntok > 0 && layer < g.n_layers && q0 + first_tok + ntok <= p.n_tokens && nt > 0 && pieces <= p.splits &&
                               key_end <= g.max_pages * g.page_size && number >= 0);
  constexpr uint32_t tmem = 0;                              // all 512 columns are this block's: they begin at 0

  float r_v = 0.f;                                          // largest V scale of the block's keys (V and softmax warps)
  // Query rows first .. of the tile at tile_tok as two e4m3 rows each, by one warp; D / 8 lanes per row, 32 / (D / 8) rows a step.  It
  // copies all of them into the place of their result (16 bytes of bf16 become 8 of the first row and 8 of the second; the lanes of
  // two neighbouring chunks write where they have read), then converts four loads at a time.
  auto stage_queries = [&](uint32_t sq, float* s_mul, int tile_tok, int first, int steps) {
    constexpr int LPR = D / 8, RPL = 32 / LPR, BATCH = 4;     // lanes per row, rows per step, steps at a time
    const int sub = lane / LPR, c8 = lane % LPR, c = c8 >> 1;   // row of the step, 8 dims of it, their 16-byte chunk of the result
    const uint32_t over_g = (65536u + G - 1) / G;             // r / G = r * over_g >> 16 for r < 128, G <= 8
    const uint32_t base = sq + (uint32_t)(c >> 3) * (kRows * 128), odd = (c8 & 1) * (uint32_t)(DH * kRows * 128);
    const int last_row = min(per_tile, ntok - tile_tok) * G;  // rows from here on are no token's
    const uint16_t* q0_ptr = p.q + (out_row0 + (long long)tile_tok * g.h_q) * D + c8 * 8;
#pragma unroll 4
    for (int i = 0; i < steps; ++i) {
      const int r = first + i * RPL + sub, rt = (int)(r * over_g >> 16);
      const uint16_t* from = r < last_row ? q0_ptr + (rt * g.h_q + (r - rt * G)) * D : p.q;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + r * 128 + (((c & 7) ^ (r & 7)) << 4) + odd), "l"(from), "r"(r < last_row ? 16 : 0) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
#pragma unroll 1
    for (int i0 = 0; i0 < steps; i0 += BATCH) {
      uint32_t w[BATCH][4], top[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = first + (i0 + i) * RPL + sub;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i][0]), "=r"(w[i][1]), "=r"(w[i][2]), "=r"(w[i][3])
                     : "r"(base + r * 128 + (((c & 7) ^ (r & 7)) << 4) + odd));
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i)   // the largest |q| of the row: bf16 magnitudes compare as integers
        top[i] = __vmaxu2(__vmaxu2(w[i][0] & 0x7FFF7FFFu, w[i][1] & 0x7FFF7FFFu), __vmaxu2(w[i][2] & 0x7FFF7FFFu, w[i][3] & 0x7FFF7FFFu));
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < BATCH; ++i) top[i] = __vmaxu2(top[i], __shfl_xor_sync(0xffffffffu, top[i], off));
      __syncwarp();                                         // both lanes of a chunk have read
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = first + (i0 + i) * RPL + sub;
        int ex = (int)(max(top[i] & 0xFFFFu, top[i] >> 16) >> 7);
        ex = ex < 8 ? 8 : (ex > 253 ? 253 : ex);
        const float down = __uint_as_float((uint32_t)(261 - ex) << 23);   // brings the largest |q| into [128, 256)
        if (c8 == 0) s_mul[r] = __uint_as_float((uint32_t)(ex - 7) << 23) * p.score_scale;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x0 = __uint_as_float(w[i][2 * e] << 16) * down, x1 = __uint_as_float(w[i][2 * e] & 0xFFFF0000u) * down;
          const float x2 = __uint_as_float(w[i][2 * e + 1] << 16) * down, x3 = __uint_as_float(w[i][2 * e + 1] & 0xFFFF0000u) * down;
          const float h0 = e4m3_head(x0), h1 = e4m3_head(x1), h2 = e4m3_head(x2), h3 = e4m3_head(x3);
          hi[e] = pack_e4m3x2(h0, h1) | (pack_e4m3x2(h2, h3) << 16);
          lo[e] = pack_e4m3x2(x0 - h0, x1 - h1) | (pack_e4m3x2(x2 - h2, x3 - h3) << 16);
        }
        const uint32_t at = base + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (c8 & 1) * 8;
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(hi[0]), "r"(hi[1]) : "memory");
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + DH * kRows * 128), "r"(lo[0]), "r"(lo[1]) : "memory");
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(qready);
  };

  if (warp >= kTma) regs_down<P::REGS_OTHER>();
  if (warp == kTma) {
    // ================= K tiles; pages and scales of their keys =================
    // Lane i < 8 looks after the tile's keys 16 i .. 16 i + 15.  A page's number and then its scales are two dependent loads, so
    // they run ahead: pages by four tiles, scales by three; they are published two tiles ahead of the K copy (the V warps
    // start from them).  A slot of the ring of kInfo tiles is free by then: K tile j is copied after S(j - KST), i.e. after the
    // softmax of tile j - KST - 2 and the V units of tile j - KST - 2, and j - KST - 2 >= j + 2 - kInfo.
    static_assert(kInfo >= KST + 4, "info ring");
    int issued = 0, vissued = 0;
    bool ok = true;
    auto page_at = [&](int j) -> int {
      const int key = (j0 + j) * kKeys + lane * 16;
      if (lane >= 8 || j >= nt || key >= key_end) return -2;   // no key
      B200ATTN_CHECK(p.status, key >= 0 && (key >> p.page_shift) < g.max_pages);
      return max(-1, ld(p.page_table + (long long)b * g.max_pages + (key >> p.page_shift)));
    };
    auto scales_at = [&](int id) -> float2 {
      if (id == -2) return make_float2(0.f, 0.f);
      if (id < 0 || id >= g.n_pages) return make_float2(-1.f, 0.f);
      const long long si = ((long long)layer * g.n_pages + id) * g.h_kv + h;
      return make_float2(ld(p.k_scale + si), ld(p.v_scale + si));
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
    int idp = -2, id0 = page_at(0), id1 = page_at(1), id2 = page_at(2), id3 = page_at(3);
    float2 sc0 = scales_at(id0), sc1 = scales_at(id1), sc2 = scales_at(id2);
    for (int j = 0; j <= nt && ok; ++j) {                   // K tile j, then V tile j - 1
      int id4_ = -2;
      float2 sc3_ = make_float2(0.f, 0.f);
      if (j < nt) {
        const int st = j % KST;
        const int id4 = page_at(j + 4);
        const float2 sc3 = scales_at(id3);
        if (j >= KST) ok = wait_for(kempty + 8 * st, ((j / KST) - 1) & 1, gave_up, p.status);
        __syncwarp();
        if (!ok) break;
        // the lane of a page's first key copies the page
        const bool box = id0 >= 0 && id0 < g.n_pages && ((lane * 16) & (g.page_size - 1)) == 0;
        const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, box));
        if (lane == 0) mbar_arrive_expect_tx(kfull + 8 * st, boxes * g.page_size * D);
        __syncwarp();
        if (box) {
          B200ATTN_CHECK(p.status, rows_exist(g, (long long)(id0 * g.h_kv + h) << p.page_shift, g.page_size, layer) && lane * 16 + g.page_size <= kKeys);
#pragma unroll
          for (int hf = 0; hf < DH; ++hf)
            tma_load_3d(sK + st * P::KTILE + hf * kKeys * 128 + lane * 16 * 128, &kmap, hf * 128, (id0 * g.h_kv + h) << p.page_shift, layer, kfull + 8 * st);
        }
        ++issued;
        if (j == 0) { publish(0, id0, sc0); publish(1, id1, sc1); }
        publish(j + 2, id2, sc2);
        id4_ = id4; sc3_ = sc3;
      }
      if (j > 0) {
        // V bytes, a unit at a time; a page of 128 keys makes two boxes where the unit has 64
        constexpr int UL = P::UNIT_KEYS / 16;               // lanes of a unit
        const int vrows = min(g.page_size, P::UNIT_KEYS);
#pragma unroll 1
        for (int u = 0; u < P::UNITS && ok; ++u) {
          const int vs = vissued % P::RAW;
          if (vissued >= P::RAW) ok = wait_for(rempty + 8 * vs, ((vissued / P::RAW) - 1) & 1, gave_up, p.status);
          __syncwarp();
          if (!ok) break;
          const bool vbox = lane / UL == u && idp >= 0 && idp < g.n_pages && ((lane * 16) & (vrows - 1)) == 0;
          const uint32_t vboxes = __popc(__ballot_sync(0xffffffffu, vbox));
          if (lane == 0) mbar_arrive_expect_tx(rfull + 8 * vs, vboxes * vrows * D);
          __syncwarp();
          if (vbox) {
            const int row = ((idp * g.h_kv + h) << p.page_shift) + ((lane * 16) & (g.page_size - 1));
            B200ATTN_CHECK(p.status, rows_exist(g, row, vrows, layer) && (lane % UL) * 16 + vrows <= P::UNIT_KEYS);
#pragma unroll
            for (int hf = 0; hf < DH; ++hf)
              tma_load_3d(sRaw + vs * P::RAW_BYTES + hf * P::UNIT_KEYS * 128 + (lane % UL) * 16 * 128, &vmap, hf * 128, row, layer, rfull + 8 * vs);
          }
          ++vissued;
        }
      }
      idp = id0; id0 = id1; id1 = id2; id2 = id3; id3 = id4_;
      sc2 = sc3_;
    }
    if (lane == 0) { s_info[8] = issued; s_info[9] = vissued; }
    __syncwarp();
    asm volatile("bar.arrive 3, %0;" ::"n"((kSoftmaxWarps + 2) * 32) : "memory");
  } else if (warp == kMma) {
    // ================= products =================
    tmem_alloc(smem_u32(s_info + 3), 512);                  // used by others only after this warp's first product
    wait_for(qready, 0, gave_up, p.status);
    __syncwarp();
    const uint32_t lowQ = (sQ >> 4) | (1u << 16), lowK = (sK >> 4) | (1u << 16), lowV = (sV >> 4) | ((uint32_t)(P::UNIT_KEYS * 128 >> 4) << 16);
    // One lane runs the whole loop.  What stands between two products leaves the tensor cores idle, so nothing is waited for twice
    // and a wait that ran out is only looked at by the waits that follow (they return at once; the results go nowhere).
    // Item n of a group is its n-th key tile: with two query tiles every key tile is one of both groups, with one the groups take
    // them in turn; heads of 256 have one group and use the two score buffers in turn.
    if (elect_one()) {
      // keys [64 sub, 64 sub + 64) of tile t (heads of 128) or all of it
      auto issue_s = [&](int t, int sub, int grp, int buf, uint32_t qa, bool wait_k, bool last) {
        const int st = t % KST;
        if (wait_k) wait_for(kfull + 8 * st, (t / KST) & 1, gave_up, p.status);
        tc_fence_after();
        const uint32_t kb0 = lowK + (uint32_t)st * (P::KTILE >> 4) + (uint32_t)sub * (8192 >> 4);
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int hf = 0; hf < DH; ++hf)
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
              umma_s(tmem + (uint32_t)(grp * 128 + buf * P::SK), qa + (term * DH + hf) * (kRows * 128 >> 4) + kb * 2, kb0 + hf * (kKeys * 128 >> 4) + kb * 2, kIdescS, (term | hf | kb) != 0);
        umma_commit(sfull + 8 * (2 * grp + buf));
        if (last) umma_commit(kempty + 8 * st);
      };
      auto issue_o = [&](int t, int half, int grp, uint32_t a, int bar, uint32_t parity, bool fresh, bool wait_v, bool last) {
        const int vu = t * P::UNITS + (P::UNITS == 2 ? half : 0), st = vu % kVRing;
        if (wait_v) wait_for(vfull + 8 * st, (vu / kVRing) & 1, gave_up, p.status);
        wait_for(pfull + 8 * bar, parity, gave_up, p.status);
        tc_fence_after();
        const uint32_t v0 = lowV + (uint32_t)st * (kUnitBytes >> 4) + (P::UNITS == 2 ? 0u : (uint32_t)half * (8192 >> 4));
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) umma_o(tmem + 256u + (uint32_t)grp * 128u, a + kb * 8, v0 + kb * (2048 >> 4), kIdescO, kb ? true : !fresh);
        umma_commit(odone + 8 * bar);
        if (last) umma_commit(vempty + 8 * st);
      };
      const uint32_t q1 = lowQ + (two ? (uint32_t)(P::QTILE >> 4) : 0u);
      if (NS == 1) {
        issue_s(0, 0, 0, 0, lowQ, true, true);
        if (nt > 1) issue_s(1, 0, 0, 1, lowQ, true, true);
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
          const int buf = t & 1;
          issue_o(t, 0, 0, tmem + buf * 128u, 2 * buf, (t >> 1) & 1, t == 0, true, true);
          issue_o(t, 1, 0, tmem + buf * 128u + 32u, 2 * buf + 1, (t >> 1) & 1, false, true, true);
          if (t + 2 < nt) issue_s(t + 2, 0, 0, buf, lowQ, true, true);
        }
      } else if (two) {
        issue_s(0, 0, 0, 0, lowQ, true, false);
        issue_s(0, 0, 1, 0, q1, false, false);
        issue_s(0, 1, 0, 1, lowQ, false, false);
        issue_s(0, 1, 1, 1, q1, false, true);
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
          const bool more = t + 1 < nt;
          issue_o(t, 0, 0, tmem, 0, t & 1, t == 0, true, false);
          if (more) issue_s(t + 1, 0, 0, 0, lowQ, true, false);
          issue_o(t, 0, 1, tmem + 128u, 2, t & 1, t == 0, false, false);
          if (more) issue_s(t + 1, 0, 1, 0, q1, false, false);
          issue_o(t, 1, 0, tmem + 64u, 1, t & 1, false, false, false);
          if (more) issue_s(t + 1, 1, 0, 1, lowQ, false, false);
          issue_o(t, 1, 1, tmem + 192u, 3, t & 1, false, false, true);
          if (more) issue_s(t + 1, 1, 1, 1, q1, false, true);
        }
      } else {
        for (int grp = 0; grp < 2; ++grp)
          if (grp < nt) { issue_s(grp, 0, grp, 0, lowQ, true, false); issue_s(grp, 1, grp, 1, lowQ, false, true); }
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
          const int grp = t & 1;
          const bool more = t + 2 < nt;
          issue_o(t, 0, grp, tmem + grp * 128u, 2 * grp, (t >> 1) & 1, t < 2, true, false);
          if (more) issue_s(t + 2, 0, grp, 0, lowQ, true, false);
          issue_o(t, 1, grp, tmem + grp * 128u + 64u, 2 * grp + 1, (t >> 1) & 1, false, false, true);
          if (more) issue_s(t + 2, 1, grp, 1, lowQ, false, true);
        }
      }
    }
    __syncwarp();
    // every softmax warp has read its output, and the TMA warp has said what it issued
    asm volatile("bar.sync 3, %0;" ::"n"((kSoftmaxWarps + 2) * 32) : "memory");
    if (*gave_up && lane == 0) {
      // A wait ran out: wait (bounded) for what was issued into this block's shared and tensor memory.
      auto drain = [&](uint32_t bar, int ring, int n) {
        for (int s = 0; s < ring && s < n; ++s) {
          const int last = ((n - 1 - s) / ring) * ring + s;
          const unsigned long long t0 = global_timer_ns();
          while (!mbar_try_wait(bar + 8 * s, (last / ring) & 1) && global_timer_ns() - t0 < kWaitBudgetNs) {}
        }
      };
      drain(kfull, KST, s_info[8]);
      drain(rfull, P::RAW, s_info[9]);
      for (int buf = 0; buf < 2; ++buf) {                   // every product was issued
        const int n = two ? nt : (nt - buf + 1) >> 1;
        for (int sub = 0; sub < NS; ++sub) drain(sfull + 8 * (NS == 2 ? 2 * buf + sub : buf), 1, n);
        drain(odone + 8 * (2 * buf + 1), 1, n);
      }
    }
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  } else if (warp >= kFirstV && warp < kTma) {
    // ================= V: bytes to f16, shared memory to shared memory =================
    regs_down<P::REGS_OTHER>();
    const int vw = warp - kFirstV, vt = tid - kFirstV * 32;
    if (NS == 1) stage_queries(sQ, s_rowmul[0], 0, vw * 32 + 16, 16 / (256 / D));   // heads of 256: half of the query rows (all of them by four warps: 3 us more)
    // the largest V scale of the block's keys
    {
      float r = kLeastV;
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
    const float inv_r = kVUp / r_v;
    // A lane's 16 bytes: chunk k4 of 64-dim block blk of a row.  Eight lanes that go together take 4 chunks of rows q and q ^ 5 of
    // an 8-row group: with both layouts swizzled (16-byte chunk index xor row) neither their loads nor their stores share a bank.
    const int k4 = lane & 3, rb = (lane >> 2) & 1, blk = D == 128 ? (lane >> 3) & 1 : lane >> 3;
    const int pr = D == 128 ? vw * 2 + (lane >> 4) : vw;    // row pair of the first step: pair 4 g + q = rows 8 g + q, 8 g + (q ^ 5)
    const int row0 = (pr >> 2) * 8 + ((pr & 3) ^ (rb ? 5 : 0));
    constexpr int STEP = D == 128 ? 16 : 8;                 // rows of one step of the four warps
    constexpr int N = P::UNIT_KEYS / STEP;                  // steps of a unit: 8
    const uint32_t src = sRaw + (D == 128 ? 0 : (blk >> 1) * (P::UNIT_KEYS * 128)) + row0 * 128 + ((((D == 128 ? blk : blk & 1) * 4 + k4) ^ (row0 & 7)) << 4);
    const uint32_t dst = sV + blk * (P::UNIT_KEYS * 128) + row0 * 128;
    const uint32_t dst0 = dst + (((2 * k4) ^ (row0 & 7)) << 4), dst1 = dst + (((2 * k4 + 1) ^ (row0 & 7)) << 4);
    const int units = nt * P::UNITS;
    bool alive = true;
#pragma unroll 1
    for (int u = 0; u < units && alive; ++u) {
      const int t = u / P::UNITS, rs = u % P::RAW, st = u % kVRing;
      alive = wait_for(kinfo + 8 * (t % kInfo), (t / kInfo) & 1, gave_up, p.status);
      if (alive) alive = wait_for(rfull + 8 * rs, (u / P::RAW) & 1, gave_up, p.status);
      if (alive && u >= kVRing) alive = wait_for(vempty + 8 * st, ((u / kVRing) - 1) & 1, gave_up, p.status);
      if (!alive) break;
      // Lane c holds the multiplier of the unit's keys 16 c ..: the page's scale relative to the largest, as an f16, and what that
      // rounds away.  Nothing is rounded where scales are powers of two (the append's): then one product per pair of values.
      const int c0 = (u % P::UNITS) * (P::UNIT_KEYS / 16), cl = c0 + lane % (P::UNIT_KEYS / 16);
      const float ratio = s_vs[t % kInfo][cl] * inv_r;
      const __half2 hi2 = __float2half2_rn(ratio), lo2 = __float2half2_rn(ratio - __low2float(hi2));
      const uint32_t hi_bits = *reinterpret_cast<const uint32_t*>(&hi2), lo_bits = *reinterpret_cast<const uint32_t*>(&lo2);
      const bool page_ok = s_id[t % kInfo][cl] >= 0;
      const int left = key_end - (j0 * kKeys + u * P::UNIT_KEYS);   // keys of the unit that exist
      const bool plain = __all_sync(0xffffffffu, page_ok && __low2float(lo2) == 0.f) && left >= P::UNIT_KEYS;
      const uint32_t pages_ok = __ballot_sync(0xffffffffu, page_ok);
#pragma unroll
      for (int i0 = 0; i0 < N; i0 += 4) {
        uint4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = lds128(src + rs * P::RAW_BYTES + (i0 + i) * STEP * 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = (i0 + i) * STEP / 16;
          const uint32_t mh = __shfl_sync(0xffffffffu, hi_bits, c);
          const __half2 hi = *reinterpret_cast<const __half2*>(&mh);
          uint32_t o[8];
          if (plain) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t h2 = e4m3x2_to_f16x2((uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu));
              const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h2), hi);
              o[e] = *reinterpret_cast<const uint32_t*>(&y);
            }
          } else {   // nothing behind the last key (bytes there may be NaN patterns), nothing of a page that does not exist
            const uint32_t ml = __shfl_sync(0xffffffffu, lo_bits, c);
            const __half2 lo = *reinterpret_cast<const __half2*>(&ml);
            const bool there = row0 + (i0 + i) * STEP < left && ((pages_ok >> c) & 1u);
            const uint32_t w[4] = {there ? raw[i].x : 0u, there ? raw[i].y : 0u, there ? raw[i].z : 0u, there ? raw[i].w : 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t h2 = e4m3x2_to_f16x2((uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu));
              const __half2 x = *reinterpret_cast<const __half2*>(&h2);
              const __half2 y = there ? __hfma2(x, hi, __hmul2(x, lo)) : x;
              o[e] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
          const uint32_t off = st * kUnitBytes + (i0 + i) * STEP * 128;
          sts128(dst0 + off, o[0], o[1], o[2], o[3]);
          sts128(dst1 + off, o[4], o[5], o[6], o[7]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(vfull + 8 * st);
        mbar_arrive(rempty + 8 * rs);
      }
    }
  } else if (warp < kSoftmaxWarps) {
    // ================= softmax: one thread per query row =================
    const int grp = warp >> 2, row = tid & 127;
    const int tile_tok = two ? grp * per_tile : 0, tok = tile_tok + row / G, head = row % G;
    const bool real = row / G < per_tile && tok < ntok;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    regs_up<P::REGS_SOFTMAX>();
    // The query rows: 32 for a warp; 16 where two groups share a tile, or the V warps take the other half.  Every thread then picks up
    // the multiplier of its own row.
    const bool halves = NS == 2 && !two;
    float rowmul;
    {
      float* s_mul = s_rowmul[two ? grp : 0];
      stage_queries(sQ + (two ? grp * P::QTILE : 0), s_mul, tile_tok, halves ? warp * 16 : (warp & 3) * 32, (halves || NS == 1 ? 16 : 32) / (256 / D));
      if (halves) asm volatile("bar.sync 1, 256;" ::: "memory");
      if (NS == 1) wait_for(qready, 0, gave_up, p.status);    // the V warps' rows
      rowmul = s_mul[row];
    }
    // keys this row sees; rows of no token see all of them (their results go nowhere, and they need no mask)
    const int vis = !real ? 0x7fffffff : p.causal ? min(len, max(0, len - nq + first_tok + tok + 1)) : len;

    float m = -INFINITY, l = 0.f;
    bool alive = true;
    const int items = two ? 2 * nt : nt;
    for (int i = grp; i < items && alive; i += NS) {
      const int j = two ? i >> 1 : i, base = (j0 + j) * kKeys;
      alive = wait_for(kinfo + 8 * (j % kInfo), (j / kInfo) & 1, gave_up, p.status);
      if (NS == 1 && alive) alive = wait_for(sfull + 8 * (i & 1), (i >> 1) & 1, gave_up, p.status);
      __syncwarp();
      if (!alive) break;
      tc_fence_after();
      const uint32_t ts = tmem + lane_base + (uint32_t)(i & 1) * 128u;
      const bool open = __all_sync(0xffffffffu, vis >= base + kKeys);   // no row of the warp has a hidden key in the tile
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {                // 64 keys at a time
        const float4 ks = *reinterpret_cast<const float4*>(s_ks[j % kInfo] + 4 * part);
        const bool bad = fminf(fminf(ks.x, ks.y), fminf(ks.z, ks.w)) < 0.f;   // a page that does not exist
        // multipliers of 16 scores each; never 0: a hidden score (-inf) times its multiplier stays -inf
        const float f[4] = {fmaxf(ks.x * rowmul, 1e-37f), fmaxf(ks.y * rowmul, 1e-37f), fmaxf(ks.z * rowmul, 1e-37f), fmaxf(ks.w * rowmul, 1e-37f)};
        const uint32_t ss = ts + 64u * part;
        if (NS == 2) {
          alive = wait_for(sfull + 8 * (2 * grp + part), (i >> 1) & 1, gave_up, p.status);
          __syncwarp();
          if (!alive) break;
          tc_fence_after();
        }
        uint32_t x[64], pk[32];
        float u;
        // Exponentials against the reference as it stands; their sum tells whether f16 can hold them.  all_exact: none by polynomial, which
        // would make a hidden score 2^-126 and a NaN a large number.
        auto exponentials = [&](auto all_exact) {
          const float mb = kBitsP - (m == -INFINITY ? 0.f : m);
          const unsigned long long mb2 = pair2(mb, mb);
          unsigned long long sum0 = 0ull, sum1 = 0ull;
#pragma unroll
          for (int e = 0; e < 64; e += 4) {
            const unsigned long long f2 = pair2(f[e >> 4], f[e >> 4]);
            float x0, x1, x2, x3;
            split2(fma2(pair2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2, mb2), x0, x1);
            split2(fma2(pair2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), f2, mb2), x2, x3);
            x0 = ex2(x0); x1 = ex2(x1);
            if (!decltype(all_exact)::value && (e / 4) % kPolyEvery == kPolyEvery - 1) {   // a share of them on the FMA pipe
              ex2_pair(x2, x3);
            } else {
              x2 = ex2(x2); x3 = ex2(x3);
            }
            sum0 = add2(sum0, pair2(x0, x1));
            sum1 = add2(sum1, pair2(x2, x3));
            const __half2 h0 = __floats2half2_rn(x0, x1), h1 = __floats2half2_rn(x2, x3);
            pk[e / 2] = *reinterpret_cast<const uint32_t*>(&h0);
            pk[e / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
          }
          float v, w;
          split2(add2(sum0, sum1), v, w);
          u = v + w;
        };
        bool fits = open && !bad && !__any_sync(0xffffffffu, m == -INFINITY);
        if (fits) {
          tmem_ld64(ss, x);
          exponentials(std::false_type());
          fits = __all_sync(0xffffffffu, u <= kMostP);       // (false for NaN)
        }
        if (!fits) {
          // Hidden keys, no reference yet, or exponentials too large or NaN: the scores again, hidden ones out, the reference to their
          // maximum if that is larger, and what O and the sum hold so far rescaled to it.
          tmem_ld64(ss, x);
          float tmax = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float kc = c == 0 ? ks.x : c == 1 ? ks.y : c == 2 ? ks.z : ks.w;
            const int seen = kc < 0.f ? 0 : vis - base - 64 * part - 16 * c;   // keys of these 16 that the row sees
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (e >= seen) x[16 * c + e] = 0xFF800000u;   // whatever the bytes there gave, NaN included
              mx = fmaxf(mx, __uint_as_float(x[16 * c + e]));
            }
            tmax = fmaxf(tmax, mx * f[c]);
          }
          float alpha = 1.f;
          if (tmax > m) {
            alpha = m == -INFINITY ? 0.f : ex2(m - tmax);
            m = tmax;
            l *= alpha;
          }
          if ((i >= NS || part) && __any_sync(0xffffffffu, alpha != 1.f)) {   // O has something in it: its last product has to be over
            if (part) alive = wait_for(odone + 8 * (2 * (i & 1)), (i >> 1) & 1, gave_up, p.status);
            else alive = wait_for(odone + 8 * (2 * ((i - NS) & 1) + 1), ((i - NS) >> 1) & 1, gave_up, p.status);
            __syncwarp();
            if (!alive) break;
            tc_fence_after();
            const uint32_t to = tmem + lane_base + 256u + (uint32_t)grp * 128u;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(to + 16 * c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16_nowait(to + 16 * c, o);
            }
          }
          exponentials(std::true_type());
        }
        l += u;
        // into the columns that the scores leave
        tmem_st32_nowait(NS == 2 ? ss : ts + 32u * part, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull + 8 * (2 * (i & 1) + part));
      }
    }

    // ---- the end: this group's last product ----
    const int mine = (items - grp + NS - 1) / NS;           // items of this group
    if (alive && mine > 0) {
      const int il = grp + (mine - 1) * NS;
      alive = wait_for(odone + 8 * (2 * (il & 1) + 1), (il >> 1) & 1, gave_up, p.status);
      __syncwarp();
      tc_fence_after();
    }
    if (halves) {
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
    if (halves) {
      const float m0 = s_ml[0][0][row], m1 = s_ml[1][0][row], l0 = s_ml[0][1][row], l1 = s_ml[1][1][row];
      M = fmaxf(m0, m1);
      f0 = m0 == -INFINITY ? l0 : ex2(m0 - M);              // no reference: the sum is 0 (no key seen) or NaN (a NaN query), and so is the weight
      f1 = m1 == -INFINITY ? l1 : ex2(m1 - M);
      L = l0 * f0 + l1 * f1;
    }
    const float unit = r_v * (1.f / kVUp), inv = pieces > 1 ? 1.f : L > 0.f ? 1.f / L : 0.f;   // two factors: unit / L can be 0 where O * unit / L is not
    float* part = p.part + ((long long)(blockIdx.x / p.splits) * p.splits + piece) * (kRows * (D + 2));
    if (alive && !*gave_up) {
#pragma unroll 1
      for (int c = halves ? grp * (D / 64) : 0; c < (halves ? (grp + 1) * (D / 64) : D / 32); ++c) {
        uint32_t x[32];
        float o[32];
        tmem_ld32(tmem + lane_base + 256u + (two ? grp * 128u : 0u) + 32 * c, x);
        tmem_wait32(x);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = f0 == 0.f ? 0.f : __uint_as_float(x[i]) * f0;
        if (halves && nt > 1) {
          tmem_ld32(tmem + lane_base + 384u + 32 * c, x);
          tmem_wait32(x);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] += f1 == 0.f ? 0.f : __uint_as_float(x[i]) * f1;
        }
        B200ATTN_CHECK(p.status, !real || (tok >= 0 && tok < ntok && head < G && row < kRows && (pieces == 1 || ((long long)(blockIdx.x / p.splits) * p.splits + piece < (long long)gridDim.x))));
        if (real && pieces == 1) {
          uint16_t* dst = p.out + (out_row0 + (long long)tok * g.h_q + head) * D + 32 * c;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const __nv_bfloat162 v2 = __floats2bfloat162_rn(o[16 * i + 2 * e] * inv * unit, o[16 * i + 2 * e + 1] * inv * unit);
              w[e] = *reinterpret_cast<const uint32_t*>(&v2);
            }
            stg256(dst + 16 * i, w);
          }
        } else if (real) {
          float4* dst = reinterpret_cast<float4*>(part + (long long)row * D + 32 * c);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float4 sums;
            sums.x = o[4 * i] * kPUnit * unit; sums.y = o[4 * i + 1] * kPUnit * unit; sums.z = o[4 * i + 2] * kPUnit * unit; sums.w = o[4 * i + 3] * kPUnit * unit;
            dst[i] = sums;
          }
        }
      }
      if (pieces > 1 && real && (!halves || grp == 0)) {
        part[kRows * D + row] = M;
        part[kRows * D + kRows + row] = L * kPUnit;
      }
    }
    tc_fence_before();
    asm volatile("bar.arrive 3, %0;" ::"n"((kSoftmaxWarps + 2) * 32) : "memory");
  }
}

// Joins the pieces of a query tile's keys: a block takes kJoinRows rows, a thread four dims of a row at a time, all loads of eight
// pieces in flight together.  (The last block to finish joining all rows of its tile by itself: 408 us for 20 tokens on 32768 keys,
// 24 / 4 heads of 256 in 36 pieces, against 81; 50 us with at most 24 pieces.)
constexpr int kJoinRows = 8, kJoinThreads = 128;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PrefillParams p) {
  pdl_wait();
  const int tile = (int)(blockIdx.x / (kRows / kJoinRows)), first = (int)(blockIdx.x % (kRows / kJoinRows)) * kJoinRows;
  const PrefillTile t = p.done[tile];
  B200ATTN_CHECK(p.status, t.rows <= kRows && t.pieces <= p.splits &&
                               (t.rows == 0 || t.row0 + (long long)((t.rows - 1) / p.g.group) * p.g.h_q + p.g.group <= (long long)p.g.n_layers * p.n_tokens * p.g.h_q));
  if (t.pieces < 2 || first >= t.rows) return;
  constexpr long long stride = kRows * (D + 2);
  const float* all = p.part + (long long)tile * p.splits * stride;
  const int G = p.g.group, end = min(t.rows, first + kJoinRows) * (D / 4);
  for (int i = first * (D / 4) + threadIdx.x; i < end; i += kJoinThreads) {
    const int r = i / (D / 4);
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < t.pieces; s0 += 8) {
      float m[8], l[8];
      float4 v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float* from = all + min(s0 + s, t.pieces - 1) * stride;
        m[s] = __ldcg(from + kRows * D + r);
        l[s] = __ldcg(from + kRows * D + kRows + r);
        v[s] = __ldcg(reinterpret_cast<const float4*>(from) + i);
        if (s0 + s >= t.pieces) m[s] = -INFINITY;
      }
      float Mn = M;
#pragma unroll
      for (int s = 0; s < 8; ++s) Mn = fmaxf(Mn, m[s]);
      const float keep = M == -INFINITY ? 0.f : ex2(M - Mn);
      M = Mn;
      L *= keep; acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float w = m[s] == -INFINITY ? 0.f : ex2(m[s] - M);
        L += l[s] * w;
        acc.x += v[s].x * w; acc.y += v[s].y * w; acc.z += v[s].z * w; acc.w += v[s].w * w;
      }
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), y = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>(p.out + (t.row0 + (long long)(r / G) * p.g.h_q + r % G) * D)[i % (D / 4)] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}

// Query tiles of a layer and head, at most: every sequence can have one that is not full, and has none without tokens.
long long prefill_tiles(const PagedGeometry& g, int n_tokens, int pair) {
  const int per_block = (kRows / g.group) << pair;
  const long long most = (long long)n_tokens / per_block + g.batch;
  return most < n_tokens ? most : n_tokens;
}
// Two query tiles in a block share its K copies, V conversion and V reads; where that leaves SMs without a block, one tile each.
int prefill_pair(const PagedGeometry& g, int n_tokens) {
  return g.head_dim == 128 && prefill_tiles(g, n_tokens, 1) * g.h_kv * g.n_layers >= device_sms() ? 1 : 0;
}
// Pieces of the keys: where the query tiles do not fill the GPU, as many as do, none under 4 tiles of keys and at most 24
// (20 tokens on 32768 keys, 24 / 4 heads of 256: 12 / 24 / 36 pieces 64 / 50 / 81 us).
int prefill_splits(const PagedGeometry& g, int n_tokens, int max_seq_len) {
  const long long cap = (long long)g.max_pages * g.page_size;
  const long long most = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  const long long blocks = prefill_tiles(g, n_tokens, prefill_pair(g, n_tokens)) * g.h_kv * g.n_layers;
  if (blocks < 1) return 1;
  long long want = device_sms() / blocks;
  const long long by_len = (most + 4 * kKeys - 1) / (4 * kKeys);
  if (want > by_len) want = by_len;
  return (int)(want < 1 ? 1 : want > 24 ? 24 : want);
}

}  // namespace

size_t paged_prefill_workspace_bytes(const PagedGeometry& g) {
  // tiles x pieces is at most the SM count whenever there are pieces
  const size_t many = (size_t)device_sms() * kRows * (g.head_dim + 2) * 4, few = paged_few_partial_bytes(g);
  return paged_partials_offset() + (many > few ? many : few) + (size_t)device_sms() * sizeof(PrefillTile);
}

cudaError_t launch_paged_prefill(const PagedGeometry& g, const PagedAttnArgs& a, cudaStream_t stream) {
  if (few_rows(g, a.n_tokens)) return launch_paged_few(g, a, stream);
  Geometry cache{};
  cache.n_layers = g.n_layers; cache.batch = g.n_pages; cache.h_kv = g.h_kv; cache.capacity = g.page_size; cache.head_dim = g.head_dim;
  CUtensorMap kmap, vmap;
  const int unit_keys = g.head_dim == 128 ? PrefillPlan<128>::UNIT_KEYS : PrefillPlan<256>::UNIT_KEYS;
  if (!encode_cache_map(&kmap, a.k_pages, cache, g.k_layer_stride, g.page_size) ||
      !encode_cache_map(&vmap, a.v_pages, cache, g.v_layer_stride, g.page_size < unit_keys ? g.page_size : unit_keys))
    return cudaErrorInvalidValue;
  PrefillParams p{};
  p.g = g;
  p.q = (const uint16_t*)a.q;
  p.k_scale = a.k_scale; p.v_scale = a.v_scale;
  p.page_table = a.page_table; p.seq_len = a.seq_len; p.q_start = a.q_start;
  p.n_tokens = a.n_tokens;
  p.causal = a.causal;
  p.page_shift = g.page_size == 16 ? 4 : g.page_size == 32 ? 5 : g.page_size == 64 ? 6 : 7;
  p.pair = prefill_pair(g, a.n_tokens);
  p.tiles = (int)prefill_tiles(g, a.n_tokens, p.pair);
  p.splits = prefill_splits(g, a.n_tokens, a.max_seq_len);
  p.score_scale = a.softmax_scale * kLog2e;
  p.part = paged_partials(a.workspace);
  p.done = (PrefillTile*)(p.part + (size_t)device_sms() * kRows * (g.head_dim + 2));   // tiles x pieces is at most the SM count
  p.out = (uint16_t*)a.out;
  p.status = a.status;
  const long long grid = (long long)p.tiles * p.splits * g.h_kv * g.n_layers;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  auto launch = [&](auto kernel, auto join, int threads, int smem) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = launch_pdl(kernel, (int)grid, threads, (size_t)smem, stream, kmap, vmap, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_pdl(join, (int)(grid / p.splits * (kRows / kJoinRows)), kJoinThreads, 0, stream, p);
  };
  return g.head_dim == 128 ? launch(paged_prefill_kernel<128>, paged_join_kernel<128>, PrefillPlan<128>::THREADS, PrefillPlan<128>::SMEM)
                           : launch(paged_prefill_kernel<256>, paged_join_kernel<256>, PrefillPlan<256>::THREADS, PrefillPlan<256>::SMEM);
}

}  // namespace b200attn
