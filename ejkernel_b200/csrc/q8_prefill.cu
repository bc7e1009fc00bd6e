// Prefill tiles over the 8-bit cache on tcgen05 + TMEM: sequences with many query rows.
//
//     S[128 x 64] = Q[128 x D] . Kc^T,   P = 2^(S * k_scale * scale * log2 e - m),   O += P . (Vc * v_scale / v_ref)
//
// The tiles, barriers, KV split and epilogue are those of rpa_prefill_sm100.cu: two 128-row tiles per CTA, 64-token stages, S and
// P.V issued by single threads, one softmax thread per row.
// What the codes add is a pipeline in front:
//
//   producer warp --raw stage (codes: bulk copies; scales: 4-byte cp.async)--> four converter warps --16-bit stage--> MMAs
//
//   * the converters write K and V as f16 (K exactly) in the swizzled layout that the tensor cores read.  An 8-bit MMA would
//     take the codes as they are, but would need q and P in 8 bits too.
//   * bf16 queries go to f16 by a power of two per row (their largest element to [2^14, 2^15)), undone on the logits.
//   * k_scale goes into the logits: where blocks have 8 tokens or more (and neither a soft cap nor a negative scale
//     interferes) as the multiplier of the exponent's FMA, one factor per 8 columns; otherwise one per column.
//   * v_scale goes into V, where it costs the softmax threads, which bound the kernel, nothing: the converters multiply by
//     v_scale / v_ref, v_ref a power of two that keeps the products within f16: the largest v_scale met so far is taken to
//     [2^6, 2^7), and a power of two times a code is exact down to 2^-24.  When a larger scale comes, v_ref grows and the
//     softmax threads rescale O, as they do when the maximum grows.
//   * one v_ref for all rows of an item must not push what some of them see out of f16: where a scale of the stage is
//     2^-11 and less of the largest one met so far ("far" stages: the mask can hide that one from a row), V goes to shared memory as
//     codes alone, and each softmax thread puts v_scale into its weights, under a power of two of its own row.  O then is in
//     units of the row's; the next common stage takes it to v_ref's.
//   * P is f16.  Its reference sits 2^7 below the maximum it was chosen for, which puts the weights between 2^15 and 2^-24:
//     what is below 2^-31 of the largest weight is lost.
//   * registers: 16 warps have 128 registers a thread; the issuing warps and the converters give theirs to the softmax
//     warps (setmaxnreg: 72 + 72 + 2 * 184 = 4 * 128).
//
// What bounds it: neither the tensor pipe nor the exponentials (0.37 busy each; float and integer instructions 0.45, issue slots 0.53)
// but the softmax threads' instructions and the instruction cache that five roles share.  4 chunks of 1740 to 1995 rows over 2136
// to 6000 keys, 32 heads over 8 kv heads of 128 (360 GFLOP): 498 us = 0.72 PFLOP/s; int8 codes 526, scale blocks of 4 tokens 560, pages
// of 24 tokens 517, a soft cap 808, head_dim 64 412, all stages far 1490.  4 sequences of 2048 rows over 8192 keys each: 1.11 ms.
// On the way there (a batch of that kind, ms): all of a stage unrolled in the converters 2.57, a rolled loop 1.73, no rare paths in
// the common kernel and paired float32 instructions 1.49, no turns between the tiles at the exponentials (which the 16-bit kernel gains
// from) 1.39, a planner of its own 1.34; the end of an item out of the loop of its stages another 2 to 6 %.  An item of one tile is
// bound by how long a stage takes to come through: 24 mixed requests with pages of 24 tokens 82 us while the producer divided for
// each page and scale, 15 to 20 % less with the stepped indexes.  Tried and dropped: two threads per row with half of the columns
// each (1.73), eight converter warps (1.46).
//
// Warp roles (512 threads, one CTA per SM, persistent over the items of q8_plan.cu):
//   warp 0 producer, warp 1 S of tile 0 (and the TMEM allocation), warp 2 S of tile 1, warp 3 P.V of all tiles,
//   warps 4-7 converters, warps 8-11 softmax of tile 0, warps 12-15 of tile 1.
//
// All hand-offs are mbarriers; every wait is bounded in wall time (Params::wait_timeout_ms): on expiry the warp raises the
// CTA's abort flag, every other wait gives up when it sees it, the status word gets EJK_RPA_ST_TIMEOUT and the CTA still
// frees its TMEM before it returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "q8_types.cuh"
#include "rpa_tcgen05.cuh"

namespace ejk {
namespace {

constexpr int kBM = kPrefillRows;  // 128 rows per tile
constexpr int kRingP = 16;
constexpr float kLog2eP = 1.4426950408889634f;
constexpr float kRefBelow = 7.0f;  // P's reference sits this far below the maximum it is chosen for ...
constexpr float kLazyP = 15.0f;    // ... and is kept until the maximum has passed it by this much: P <= 2^15 < 65504
constexpr int kVBits = 6;          // the largest v_scale met so far is taken to [2^6, 2^7): 448 * 2^7 < 65504
constexpr float kFar = 0x1p-5f;    // a stage is far where a scale is below this in those units: its smallest codes leave f16's normals
constexpr float kFarV = 0x1p7f;    // what a far stage's codes are multiplied by, and its weights divided

// One piece of work of a CTA, as in rpa_prefill_sm100.cu.
struct ItemDescP {
  Unit u;
  int32_t h;
  int32_t first_stage;  // index of the (item, head)'s first stage in the global stage sequence
  int32_t quota;        // stages per CTA
  int32_t pad;
};

template <int D>
struct CfgP {
  static constexpr int BN = 64;                       // tokens per KV stage
  static constexpr int NT = 2;                        // 128-row tiles per CTA
  static constexpr int SM_WARPS = 4;                  // softmax warps per tile: one thread per row
  static constexpr int CV_WARPS = 4;                  // converter warps
  static constexpr int THREADS = 32 * (4 + CV_WARPS + SM_WARPS * NT);
  static constexpr int REGS = 65536 / THREADS / 8 * 8;  // per thread at launch
  static constexpr int REGS_ISSUE = 72, REGS_CONVERT = 72, REGS_SOFTMAX = 184;
  static_assert(REGS_ISSUE + REGS_CONVERT + NT * REGS_SOFTMAX <= (2 + NT) * REGS, "setmaxnreg.inc draws on the block's own registers");
  static constexpr int RAW_BYTES = BN * 2 * D;        // a stage of codes: [K|V][BN][D]
  static constexpr int STAGE_BYTES = BN * 2 * D * 2;  // a stage of 16-bit values
  // 16-bit stages and stages of codes: what shared memory holds beside the query tiles
  static constexpr int NS = (D == 64) ? 6 : 3;
  static constexpr int NR = (D == 64) ? 4 : 3;
  static constexpr int GROUP_BYTES = 8 * 2 * D * 2;   // one 8-token group of a 16-bit stage: [K|V][D/64][8][64]
  static constexpr int V_OFF = (D / 64) * 1024;
  static constexpr int Q_BYTES = kBM * D * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = OFF_Q + NT * Q_BYTES;
  static constexpr int OFF_RAW = OFF_KV + NS * STAGE_BYTES;
  static constexpr int OFF_RAWSCALE = OFF_RAW + NR * RAW_BYTES;      // per raw stage: BN scales of K, BN of V (at most)
  static constexpr int OFF_KSCALE = OFF_RAWSCALE + NR * 2 * BN * 4;  // per 16-bit stage: each token's factor on its logits
  static constexpr int OFF_VSCALE = OFF_KSCALE + NS * BN * 4;        // per far stage: each token's V scale
  static constexpr int OFF_RING = OFF_VSCALE + NS * BN * 4;
  static constexpr int OFF_RMETA = OFF_RING + kRingP * (int)sizeof(ItemDescP);
  static constexpr int OFF_META = OFF_RMETA + NR * 8;
  static constexpr int OFF_VREF = OFF_META + NS * 8;                 // per 16-bit stage: 1 / v_ref, negative: a far stage
  static constexpr int OFF_BAR = (OFF_VREF + NS * 4 + 7) / 8 * 8;
  // barriers: kv_full[NS] kv_empty[NS] raw_full[NR] raw_empty[NR], then per tile: s_full s_free p_full[2] pv_done[2]
  // q_full o_free
  static constexpr int BAR_PER_TILE = 8;
  static constexpr int N_BAR = 2 * NS + 2 * NR + NT * BAR_PER_TILE;
  static constexpr int OFF_TMEM = OFF_BAR + N_BAR * 8;
  // abort flag, the published-items counter, per tile the count of items its softmax warps have skipped
  static constexpr int OFF_ABORT = OFF_TMEM + 8;
  static constexpr int SMEM_BYTES = OFF_ABORT + 8 + 4 * NT + 1024;
  static constexpr uint32_t P_COLS = BN / 2;               // one P buffer (16-bit pairs)
  static constexpr uint32_t TMEM_S = 0;                    // S_x at x*BN
  static constexpr uint32_t TMEM_P = NT * BN;              // P_x[b] at 2*BN + (2x + b)*P_COLS
  static constexpr uint32_t TMEM_O = 512 - NT * D;         // O_x at the top
  static constexpr uint32_t TMEM_COLS = 512;
  static_assert(BN % 16 == 0 && TMEM_P + NT * 2 * P_COLS <= TMEM_O, "TMEM holds 512 columns");
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// untiled bulk copy: both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
}
template <int N>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
}
// two float32 in one instruction
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, __half2 b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// A far stage of a softmax thread: what the kernel does with the others' (which see there), but with the tokens' V scales in the
// weights, under a power of two of the row's own.  Such stages are rare, and the length of the softmax warps' code bounds the
// kernel (in line, 4 prompt chunks took 543 to 585 us instead of 500), so that this is a call that works on a copy of the logits
// in local memory.
struct FarRow {
  float m, l, v;  // reference of the weights, their sum, the units of O
  bool ok;        // false: a wait ran out
};
template <int D, bool PLAIN>
__device__ __noinline__ FarRow far_stage(FarRow r, const float* kf, const float* vs, float q_fac, float cap_log2, int hi_i, int lo_i,
                                         uint32_t tm_s, uint32_t tm_p, uint32_t tm_o, uint32_t bar_s_free, uint32_t bar_p_full,
                                         uint32_t bar_pv_before, uint32_t bar_pv_last, int ti, bool first, volatile int* abort_flag,
                                         unsigned long long wait_ns) {
  constexpr int BN = CfgP<D>::BN;
  const int lane = threadIdx.x & 31;
  float y[BN], mx = -INFINITY, top = 0.f;
#pragma unroll 1
  for (int c0 = 0; c0 < BN; c0 += 16) {
    uint32_t s[16];
    tc_ld16(tm_s + c0, s);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int i = c0 + j;
      // in the common kernel the factor is one per 8 columns, and the soft cap is elsewhere
      const float f = kf[PLAIN ? i >> 3 : i] * q_fac;
      float v = __uint_as_float(s[j]) * f;
      if (!PLAIN && cap_log2 != 0.f) v = fmaf(fast_reciprocal(fast_exp2(v) + 1.f), -2.f * cap_log2, cap_log2);
      if (i > hi_i || i <= lo_i) v = -INFINITY;
      else top = fmaxf(top, vs[i]);
      mx = fmaxf(mx, v);
      y[i] = v;
    }
  }
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar_s_free);
  r.ok = ti < 2 || mbar_wait(bar_pv_before, ((ti - 2) >> 1) & 1, abort_flag, wait_ns);
  if (!r.ok) return r;
  // The row's units: its largest V scale to [2^6, 2^7).  v_ref is never above that, so the next common stage cannot ask for
  // finer units than these.
  float v_new = r.v;
  if (top > 0.f) {
    if (r.m == -INFINITY) v_new = __uint_as_float((127u + 125u) << 23);  // the row has seen no scale yet
    if (top * v_new >= (float)(2 << kVBits)) {
      uint32_t e = __float_as_uint(top) >> 23;
      e = e < 8u ? 8u : e;
      v_new = __uint_as_float((254u + kVBits - e) << 23);
    }
  }
  const bool grow = (mx > r.m + kLazyP) || (r.m == -INFINITY && mx > -INFINITY);
  if (__any_sync(0xffffffffu, grow || v_new != r.v)) {
    float alpha = r.m > -INFINITY ? v_new * power_of_two_inverse(r.v) : 1.f;
    if (grow) {
      const float f = fast_exp2(r.m - (mx - kRefBelow));
      r.m = mx - kRefBelow;
      r.l *= f;
      alpha *= f;
    }
    r.v = v_new;
    if (!first) {
      r.ok = mbar_wait(bar_pv_last, ((ti - 1) >> 1) & 1, abort_flag, wait_ns);
      if (!r.ok) return r;
      tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 16) {
        uint32_t o[16];
        tc_ld16(tm_o + c0, o);
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
        tc_st16(tm_o + c0, o);
      }
    }
  }
  const float m_use = r.m == -INFINITY ? 0.f : r.m, unit = r.v * (1.f / kFarV);
#pragma unroll 1
  for (int c0 = 0; c0 < BN; c0 += 32) {
    uint32_t pk[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int i = c0 + 2 * j;
      const float p0 = fast_exp2(y[i] - m_use), p1 = fast_exp2(y[i + 1] - m_use);
      r.l += p0 + p1;
      // a key without weight has none whatever its scale: it may be one that the row does not see
      pk[j] = Mma<__half>::pack(p0 == 0.f ? 0.f : p0 * (vs[i] * unit), p1 == 0.f ? 0.f : p1 * (vs[i + 1] * unit));
    }
    tc_st16(tm_p + (c0 >> 1), pk);
  }
  tc_wait_st();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar_p_full);
  return r;
}

// PLAIN: scale blocks of 8 tokens or more, no soft cap, a positive scale
template <typename T, typename Code, int D, bool PLAIN>
__global__ void __launch_bounds__(CfgP<D>::THREADS, 1)
q8_prefill_kernel(const Params p, const Q8Cache cache) {
  using C = CfgP<D>;
  constexpr int NS = C::NS, NR = C::NR, NT = C::NT, kBN = C::BN;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sb = smem_u32(smem);
  ItemDescP* ring = reinterpret_cast<ItemDescP*>(smem + C::OFF_RING);
  int2* metas = reinterpret_cast<int2*>(smem + C::OFF_META);
  int2* raw_metas = reinterpret_cast<int2*>(smem + C::OFF_RMETA);
  float* vrefs = reinterpret_cast<float*>(smem + C::OFF_VREF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_ABORT);
  volatile int* items_pub = reinterpret_cast<volatile int*>(smem + C::OFF_ABORT + 4);  // items in the ring so far
  // skipped[x]: one count per softmax warp of tile x and item without rows for the tile.  A counter, not an
  // mbarrier: the group is not held back by anybody while it skips items, so it can be several items
  // ahead of the role that waits for it, and a phase parity would alias.
  volatile int* skipped = reinterpret_cast<volatile int*>(smem + C::OFF_ABORT + 8);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::OFF_TMEM);
  const uint32_t bar0 = sb + C::OFF_BAR;
  auto bar_kv_full = [&](int s) { return bar0 + s * 8; };
  auto bar_kv_empty = [&](int s) { return bar0 + (NS + s) * 8; };
  auto bar_raw_full = [&](int s) { return bar0 + (2 * NS + s) * 8; };
  auto bar_raw_empty = [&](int s) { return bar0 + (2 * NS + NR + s) * 8; };
  auto tile_bar = [&](int x, int i) { return bar0 + (2 * NS + 2 * NR + x * C::BAR_PER_TILE + i) * 8; };
  auto bar_s_full = [&](int x) { return tile_bar(x, 0); };    // S_x(t) complete (commit)
  auto bar_s_free = [&](int x) { return tile_bar(x, 1); };    // S_x(t) is in the 4 warps' registers
  auto bar_p_full = [&](int x, int b) { return tile_bar(x, 2 + b); };   // P_x(t) stored to buffer t&1 by the softmax warps
  auto bar_pv_done = [&](int x, int b) { return tile_bar(x, 4 + b); };  // P_x.V(t) complete (commit): buffer t&1 is free
  auto bar_q_full = [&](int x) { return tile_bar(x, 6); };
  auto bar_o_free = [&](int x) { return tile_bar(x, 7); };

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int Hkv = p.Hkv, G = p.G;
  const unsigned long long wait_ns = (unsigned long long)p.wait_timeout_ms * 1000000ull;
  unsigned flags = 0;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(bar_kv_full(s), C::CV_WARPS);
      // released by the MMA-issuing roles, once per tile for S and once for P.V (commit, or a plain arrival
      // when the tile is idle)
      mbar_init(bar_kv_empty(s), 2 * NT);
    }
    for (int s = 0; s < NR; ++s) {
      mbar_init(bar_raw_full(s), 1 + 32);  // the announcement, and every producer lane's scale copies
      mbar_init(bar_raw_empty(s), C::CV_WARPS);
    }
    for (int x = 0; x < NT; ++x) {
      mbar_init(bar_s_full(x), 2);  // the commit, and the issuer's own arrival: it has seen the stage (see there)
      mbar_init(bar_s_free(x), C::SM_WARPS);  // one arrival per softmax warp
      for (int b = 0; b < 2; ++b) {
        mbar_init(bar_p_full(x, b), C::SM_WARPS);
        mbar_init(bar_pv_done(x, b), 1);
      }
      mbar_init(bar_q_full(x), C::SM_WARPS);
      mbar_init(bar_o_free(x), C::SM_WARPS);
      skipped[x] = 0;
    }
    *abort_flag = 0;
    *items_pub = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(sb + C::OFF_TMEM), "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Launched as a programmatic dependent of the planner: everything above overlapped its tail.  The
  // split-KV kernel that follows in the stream works on other rows and may start on SMs that this
  // kernel's CTAs have left; it is released once every CTA has passed this point, i.e. after the
  // plan is complete.
  if (p.pdl & 1) pdl_wait();
  pdl_trigger();
  // Mixed batch: this kernel is compute-bound, the split-KV kernel behind it bandwidth-bound, and a CTA of each does not fit
  // one SM together.  So this kernel keeps only as many CTAs as make it end about when the other does; the rest exit at
  // once and hand their SMs over (the rule of rpa_prefill_sm100.cu).
  int n_cta = (int)gridDim.x;
  if ((p.pdl & 1) && p.prefill_share > 0) {
    const float stages = (float)p.header[kHdrPrefillStages] * (float)Hkv;           // (item, head) stages of 64 tokens
    const float dec_bytes = (float)p.header[kHdrTotalKeys] * (float)Hkv * (float)(2 * D);
    // One stage of two 128-row tiles (also taken for items of one), and what a soft cap's tanh adds; the rate is an upper estimate
    // of the split-KV kernel's (4.8 to 6.3 TB/s), which the share above 100 makes good: 96 decode rows of 6000 keys beside 4 chunks of 512 tokens
    // 399 us at 125, 479 at 100, 569 at 75, 408 with no share taken; batches with less to decode do not depend on it
    const float kStageUs = (D == 64 ? 1.15f : 1.25f) * (p.cap != 0.f ? 1.6f : 1.f);
    constexpr float kDecodeBpUs = 6.6e6f;  // bytes per microsecond the split-KV kernel streams
    const float t_p = stages * kStageUs / (float)gridDim.x, t_d = dec_bytes / kDecodeBpUs;
    if (t_d > t_p && t_p > 0.f) {
      int n = (int)ceilf((float)gridDim.x * (t_p / t_d) * (float)p.prefill_share * 0.01f);
      const int floor_n = (int)gridDim.x / 8;
      n = n < floor_n ? floor_n : n;
      n_cta = n < (int)gridDim.x ? n : (int)gridDim.x;
    }
  }
  const bool idle_cta = (int)blockIdx.x >= n_cta;
  const int n_work = idle_cta ? 0 : p.header[kHdrNumPrefill] * Hkv;

  // the register split: every warp of a warpgroup at the same place, the shares add up to the registers that the block is
  // launched with (checked on the host)
  if (warp < 4) {
    give_registers<C::REGS_ISSUE>();
    if (warp == 0) {
    // =============================== producer ===============================
    const int pb = p.tma_block_tokens, pb_shift = p.tma_block_shift;  // tokens of a page that one copy takes
    const int sb_shift = cache.block_shift;
    const int scales_per_page = p.page_size >> sb_shift;
    const size_t plane_bytes = (size_t)p.page_size * D;
    const int step_pages = kBN / p.page_size, step_off = kBN % p.page_size;
    int gi = 0;  // stage counter of this CTA
    int k = 0;
    // Whole (item, head) pairs from the planner's longest-first queue, or, where that schedule is clearly worse, equal
    // quotas of the stages of all pairs (see rpa_prefill_sm100.cu)
    const int n_items = p.header[kHdrNumPrefill];
    const long long W = idle_cta ? 0 : (long long)p.header[kHdrPrefillStages] * Hkv;
    constexpr int kMinQuota = 8;  // a part shorter than this is all overhead
    bool split = p.prefill_split && W > 0 && W < (1ll << 30);
    long long quota_ll = (W + n_cta - 1) / n_cta;
    if (quota_ll < kMinQuota) quota_ll = kMinQuota;
    if (split && p.prefill_split < 2) {  // 2 = always split (measurement aid)
      const long long U = (long long)n_items * Hkv, Cn = n_cta;
      const long long rounds = (U + Cn - 1) / Cn;
      split = rounds * W * 20 >= 23 * U * (quota_ll + 16);  // rounds * W / U >= 1.15 * (quota + 16)
    }
    const int quota = split ? (int)quota_ll : 0;
    long long g = (long long)blockIdx.x * quota;                 // next global stage of this CTA
    const long long g_end = (g + quota < W) ? g + quota : W;
    int it = 0;                                                  // item that contains stage g
    if (split && g < g_end) {
      int lo = 0, hi = n_items;  // Hkv * pprefix[lo] <= g < Hkv * pprefix[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)Hkv * __ldg(p.pprefix + mid) <= g) lo = mid;
        else hi = mid;
      }
      it = lo;
    }
    int wid = 0;
    if (!split && !idle_cta) {  // a CTA that has handed its SM over must not draw from the queue
      if (lane == 0) wid = atomicAdd(&p.header[kHdrPrefillQueue], 1);
      wid = __shfl_sync(0xffffffffu, wid, 0);
    }
    bool alive = true;
    while (alive) {
      const int s = gi % NR;
      if (split ? (g >= g_end) : (wid >= n_work)) {
        if (!mbar_wait(bar_raw_empty(s), ((gi / NR) & 1) ^ 1, abort_flag, wait_ns)) break;
        if (lane == 0) {
          raw_metas[s] = make_int2(-1, 0);
          ring[k % kRingP].u.seq = -1;  // end of the item sequence, for the softmax groups
          __threadfence_block();
          *items_pub = k + 1;
          mbar_arrive(bar_raw_full(s));
        }
        cp_async_arrive(bar_raw_full(s));
        ++gi;
        break;
      }
      int ui, h, first_stage = 0;
      int st_b = 0, st_e = -1;  // the piece's stage range inside the item (st_e < 0: the whole item)
      int n_parts = 1, part_idx = 0;
      if (split) {
        const int p0 = __ldg(p.pprefix + it), p1 = __ldg(p.pprefix + it + 1);
        const int n_i = p1 - p0;                                  // stages of the item (per head)
        const long long rel = g - (long long)Hkv * p0;
        ui = it;
        h = (int)(rel / n_i);
        st_b = (int)(rel - (long long)h * n_i);
        const long long left = g_end - g;
        const int take = (n_i - st_b < left) ? n_i - st_b : (int)left;
        st_e = st_b + take;
        first_stage = (int)((long long)Hkv * p0 + (long long)h * n_i);
        const int c0 = first_stage / quota, c1 = (first_stage + n_i - 1) / quota;
        n_parts = c1 - c0 + 1;
        part_idx = (int)blockIdx.x - c0;
        g += take;
        if (st_e == n_i && h == Hkv - 1) ++it;
        if (st_e == n_i) st_e = -1;  // up to the item's real end (its last stage may be ragged)
      } else {
        ui = wid / Hkv;
        h = wid - ui * Hkv;
      }
      Unit u;
      {
        const int4* src = reinterpret_cast<const int4*>(p.punits + ui);
        const int4 a = __ldg(src), b = __ldg(src + 1);
        u.seq = a.x; u.row0 = a.y; u.kv_begin = a.z; u.kv_end = a.w;
        u.slot = b.x; u.q_start = b.y; u.q_len = b.z; u.kv_len = b.w;
        u.merge_idx = ui * Hkv + h; u.chunk_idx = part_idx; u.n_chunks = n_parts; u.pad = 0;
        if (st_e >= 0) u.kv_end = u.kv_begin + st_e * kBN;
        u.kv_begin += st_b * kBN;
      }
      const int ring_slot = k % kRingP;
      int wid_next = 0;
      if (!split && lane == 0) wid_next = atomicAdd(&p.header[kHdrPrefillQueue], 1);
      const int32_t* tab = p.block_tables + (size_t)u.seq * p.pages_per_seq;
      bool first = true;
      // where this lane's block of tokens lies: divided out once per item and stepped from then on; the id of a stage's page is
      // on its way while the stage before it is issued
      int pi, off;
      {
        const int key = u.kv_begin + (lane << pb_shift);
        if (p.page_shift >= 0) {
          pi = key >> p.page_shift;
          off = key & (p.page_size - 1);
        } else {
          pi = key / p.page_size;
          off = key - pi * p.page_size;
        }
      }
      auto blocks_at = [&](int pos) {
        const int n = (u.kv_end - pos + pb - 1) >> pb_shift;
        return n < 0 ? 0 : n > (kBN >> pb_shift) ? kBN >> pb_shift : n;
      };
      int id_next = lane < blocks_at(u.kv_begin) ? __ldg(tab + pi) : 0;
      for (int pos = u.kv_begin; first || pos < u.kv_end; pos += kBN) {
        const int st = gi % NR;
        const int nblk = blocks_at(pos);
        int page = id_next;
        if ((unsigned)page >= (unsigned)p.num_pages) {
          flags |= EJK_RPA_ST_PAGE_ID;
          page = 0;
        }
        const int at_off = off;
        pi += step_pages;
        off += step_off;
        if (off >= p.page_size) {
          off -= p.page_size;
          ++pi;
        }
        id_next = lane < blocks_at(pos + kBN) ? __ldg(tab + pi) : 0;
        if (!mbar_wait(bar_raw_empty(st), ((gi / NR) & 1) ^ 1, abort_flag, wait_ns)) {
          alive = false;
          break;
        }
        // test hook: the stage's data is never announced (no arrival, no copies), so the waits for it must
        // run out; the item itself is published as usual, so that every role sees a valid descriptor
        const bool withhold = (p.test_withhold & 2) && first && (split ? (blockIdx.x == 0 && k == 0) : (wid == 0));
        const uint32_t full = bar_raw_full(st);
        if (lane == 0) {
          if (first) {
            // every role is within NR + NS + 2 items of this warp (the converters and MMA warps through the stage rings, each
            // softmax group through q_full or its skip count): slot k - kRingP is free
            ItemDescP d;
            d.u = u;
            d.h = h;
            d.first_stage = first_stage;
            d.quota = quota;
            d.pad = 0;
            ring[ring_slot] = d;
            __threadfence_block();
            *items_pub = k + 1;
          }
          // meta.x = ring slot | 0x100 on the first stage of an item | 0x200 when the item has rows for tile 1
          const bool two = u.slot > kBM && u.q_len * G > u.row0 + kBM;
          raw_metas[st] = make_int2(ring_slot | (first ? 0x100 : 0) | (two ? 0x200 : 0), pos);
          const uint32_t bytes = (uint32_t)nblk * (uint32_t)pb * 2 * D;
          if (withhold) {
          } else if (bytes > 0) {
            mbar_arrive_expect_tx(full, bytes);
          } else {
            mbar_arrive(full);
          }
        }
        __syncwarp();
        if (!withhold) {
          if (lane < nblk) {
            const uint8_t* src = cache.pages + (((size_t)page * Hkv + h) * 2) * plane_bytes + (size_t)at_off * D;
            const uint32_t dst = sb + C::OFF_RAW + st * C::RAW_BYTES + (uint32_t)(lane << pb_shift) * D;
            bulk_load(dst, src, (uint32_t)pb * D, full);
            bulk_load(dst + kBN * D, src + plane_bytes, (uint32_t)pb * D, full);
          }
          // scales of the blocks that the stage's keys lie in: K's, then V's
          const int e0 = pos >> sb_shift;
          const int last = (u.kv_end < pos + kBN ? u.kv_end : pos + kBN) - 1;
          const int n_e = last >= pos ? (last >> sb_shift) - e0 + 1 : 0;
          const uint32_t sdst = sb + C::OFF_RAWSCALE + st * (2 * kBN * 4);
          for (int b0 = 0; b0 < n_e; b0 += 32) {
            const int e = b0 + lane;
            int rel = ((e0 + e) << sb_shift) - pos;  // the block's first key in the stage; its page is that of a lane's tokens
            rel = e < n_e && rel > 0 ? rel : 0;
            const int of_page = __shfl_sync(0xffffffffu, page, rel >> pb_shift);
            const int eoff = __shfl_sync(0xffffffffu, at_off, rel >> pb_shift) + (rel & (pb - 1));
            if (e < n_e) {
              const float* src = cache.scales + (((long long)of_page * Hkv + h) * 2) * scales_per_page + (eoff >> sb_shift);
              cp_async4(sdst + e * 4, src);
              cp_async4(sdst + (kBN + e) * 4, src + scales_per_page);
            }
          }
          cp_async_arrive(full);
        }
        first = false;
        ++gi;
      }
      ++k;
      if (!split) wid = __shfl_sync(0xffffffffu, wid_next, 0);
    }
    // wait (bounded) until every stage this warp filled has been released, i.e. all its bulk
    // copies have landed and been consumed
    for (int i = 0; i < NR; ++i) {
      const int g2 = gi + i;
      if (g2 < NR) continue;  // never used
      if (!mbar_wait(bar_raw_empty(g2 % NR), ((g2 / NR) & 1) ^ 1, abort_flag, wait_ns)) break;
    }
    if (*abort_flag) {
      // giving up: nobody releases stages any more, so wait (bounded, 2 ms per stage) for the copies
      // themselves -- the "full" phase of each of the last NR announced stages
      for (int i = 1; i <= NR && i <= gi; ++i) {
        const int f = gi - i;
        mbar_wait_quiet(bar_raw_full(f % NR), (uint32_t)((f / NR) & 1), 2000000ull);
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    } else {
    // =============================== MMA issuers ===============================
    // Single-thread roles, ordered by the barriers alone: S_x(t+1) needs the S columns back (s_free), P_x.V(t) needs P_x(t)
    // (p_full); both need the stage (kv_full).
    if (lane == 0) {
      const bool is_s = warp < 3;
      const int x = is_s ? warp - 1 : 0;
      constexpr uint32_t idesc_s = instr_desc<__half>(kBN, false);
      constexpr uint32_t idesc_pv = instr_desc<__half>(D, true);
      // hi word of a descriptor: stride byte offset >> 4, version 1 (bit 46), SWIZZLE_128B (bits 61-63)
      constexpr uint64_t kHiAtom1024 = ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29))) << 32;
      constexpr uint64_t kHiGroup = ((uint64_t)(((uint32_t)C::GROUP_BYTES >> 4) | (1u << 14) | (2u << 29))) << 32;
      const uint64_t q_desc = kHiAtom1024 | (uint64_t)(((sb + C::OFF_Q + x * C::Q_BYTES) >> 4) | (1u << 16));
      const uint64_t k_desc0 = kHiGroup | (uint64_t)(((sb + C::OFF_KV) >> 4) | (1u << 16));
      // V is MN-major: leading byte offset = distance between 64-element chunks of D (1024 B)
      const uint64_t v_desc0 = kHiGroup | (uint64_t)(((sb + C::OFF_KV + C::V_OFF) >> 4) | ((1024u >> 4) << 16));
      const uint32_t tm_s = tmem_base + C::TMEM_S + x * kBN;

      int gi = 0;     // KV stage counter (every role sees the same stage sequence)
      int t = 0;      // stages this tile took part in (barrier parities)
      int items = 0;  // items this tile took part in
      int skips = 0;  // items this tile had no rows for
      int tx[NT], itemsx[NT];  // the same two counters per tile, for the P.V role
#pragma unroll
      for (int y = 0; y < NT; ++y) tx[y] = itemsx[y] = 0;
      while (!is_s) {
        // ---- P.V of all tiles, tile 0 first ----
        const int st = gi % NS;
        if (!mbar_wait_thread(bar_kv_full(st), (gi / NS) & 1, abort_flag, wait_ns)) break;
        const int mx = metas[st].x;
        if (mx < 0) break;
        const bool first = (mx & 0x100) != 0;
        bool gave_up = false;
#pragma unroll
        for (int y = 0; y < NT; ++y) {
          if (gave_up) continue;
          if (y > 0 && !(mx & 0x200)) {  // no rows for this tile: only its share of the stage's release
            mbar_arrive(bar_kv_empty(st));
            continue;
          }
          if (first) ++itemsx[y];
          const int ty = tx[y];
          // O_y (+)= P_y . V: P_y(t) must be in its TMEM buffer; the first P.V of an item overwrites
          // O_y, which the previous item's epilogue must have read
          if (!mbar_wait_thread(bar_p_full(y, ty & 1), (ty >> 1) & 1, abort_flag, wait_ns) ||
              (first && itemsx[y] > 1 && !mbar_wait_thread(bar_o_free(y), itemsx[y] & 1, abort_flag, wait_ns))) {
            gave_up = true;
            continue;
          }
          tc_fence_after();
          const uint32_t tm_p = tmem_base + C::TMEM_P + y * 2 * C::P_COLS;
          const uint32_t tm_o = tmem_base + C::TMEM_O + y * D;
          const uint64_t vd = v_desc0 + (uint64_t)((st * C::STAGE_BYTES) >> 4);
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk) {
            // V: 16 tokens = two 8-token groups per MMA; P: 16 tokens = 8 columns of 16-bit pairs
            tc_mma_ts(tm_o, tm_p + (ty & 1) * C::P_COLS + kk * 8, vd + (uint64_t)((kk * 2 * C::GROUP_BYTES) >> 4), idesc_pv,
                      !(first && kk == 0));
          }
          tc_commit(bar_pv_done(y, ty & 1));
          tc_commit(bar_kv_empty(st));  // this tile's P.V MMAs that read the stage have been issued
          ++tx[y];
        }
        if (gave_up) break;
        ++gi;
      }
      while (is_s) {
        const int st = gi % NS;
        if (!mbar_wait_thread(bar_kv_full(st), (gi / NS) & 1, abort_flag, wait_ns)) break;
        const int mx = metas[st].x;
        if (mx < 0) break;
        const bool first = (mx & 0x100) != 0;
        const bool act = (x == 0) || (mx & 0x200) != 0;
        if (!act) {  // the item has no rows for this tile: only this role's share of the stage's release
          if (first) {
            // ... once the tile's softmax group has seen the item, so that it never falls behind
            ++skips;
            bool seen = skipped[x] >= C::SM_WARPS * skips;
            if (!seen) {
              const unsigned long long t0 = global_timer_ns();
              while (!(seen = skipped[x] >= C::SM_WARPS * skips)) {
                if (*abort_flag) break;
                if (global_timer_ns() - t0 > wait_ns) {
                  *abort_flag = 1;
                  break;
                }
                __nanosleep(64);
              }
            }
            if (!seen) break;
          }
          mbar_arrive(bar_kv_empty(st));
          ++gi;
          continue;
        }
        if (first) ++items;
        {
          // the new query tile must be in shared memory, and S_x of the previous stage in the
          // softmax warps' registers
          if (first && !mbar_wait_thread(bar_q_full(x), (items - 1) & 1, abort_flag, wait_ns)) break;
          if (t > 0 && !mbar_wait_thread(bar_s_free(x), (t - 1) & 1, abort_flag, wait_ns)) break;
          tc_fence_after();
          // the softmax warps read the stage's factors after waiting for S alone: this arrival, after the wait for the
          // stage, orders those reads behind the converters' writes
          mbar_arrive(bar_s_full(x));
          const uint64_t kd = k_desc0 + (uint64_t)((st * C::STAGE_BYTES) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            // K: 8-token atoms one group apart (SBO), the 64-element chunks of D 1024 bytes apart
            const uint32_t koff = (uint32_t)(((kk >> 2) * 1024 + (kk & 3) * 32) >> 4);
            const uint32_t qoff = (uint32_t)(((kk >> 2) * (kBM * 128) + (kk & 3) * 32) >> 4);
            tc_mma(tm_s, q_desc + qoff, kd + koff, idesc_s, kk > 0);
          }
          tc_commit(bar_s_full(x));
        }
        tc_commit(bar_kv_empty(st));  // this role's MMAs that read the stage have been issued
        ++t;
        ++gi;
      }
    }
    __syncwarp();
    }
  } else if (warp < 4 + C::CV_WARPS) {
    give_registers<C::REGS_CONVERT>();
    // =============================== converters ===============================
    const int ctid = tid - 128;  // 0 .. 127
    const int sb_shift = cache.block_shift;
    // Sixteen codes of a token per thread and step: a quarter warp reads 128 consecutive bytes, and writes the two 16-byte
    // halves of its 32 bytes in an order that keeps its eight stores on different banks.
    constexpr int CPT = D / 16;           // 16-code chunks per token
    constexpr int TSTEP = 128 / CPT;      // tokens per step of the four warps
    static_assert(kBN % TSTEP == 0, "whole steps");
    const int ch = ctid % CPT, t0 = ctid / CPT;
    const int half_first = D == 128 ? (ch >> 2) & 1 : 0;
    const uint32_t c_first = (uint32_t)((2 * ch + half_first) & 7), c_second = c_first ^ 1u;
    constexpr bool coarse = PLAIN;        // one factor per 8 tokens is enough
    const float to_log2 = p.cap != 0.f ? p.inv_cap_scale * (2.f * kLog2eP) : p.scale_log2;
    float v_norm = 1.f;
    int lo_min = -1, kv_end = 0;
    int gi = 0;
    while (true) {
      const int rs = gi % NR, st = gi % NS;
      if (!mbar_wait(bar_raw_full(rs), (gi / NR) & 1, abort_flag, wait_ns)) break;
      const int2 meta = raw_metas[rs];
      if (meta.x < 0) {  // the end marker goes on
        if (!mbar_wait(bar_kv_empty(st), ((gi / NS) & 1) ^ 1, abort_flag, wait_ns)) break;
        if (ctid == 0) metas[st] = meta;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_kv_full(st));
          mbar_arrive(bar_raw_empty(rs));
        }
        break;
      }
      const int pos = meta.y;
      const float* ks_s = reinterpret_cast<const float*>(smem + C::OFF_RAWSCALE + rs * (2 * kBN * 4));
      const float* vs_s = ks_s + kBN;
      const int e0 = pos >> sb_shift;
      if (meta.x & 0x100) {
        const Unit& u = ring[meta.x & 0xff].u;
        kv_end = u.kv_end;
        lo_min = (p.window > 0) ? (u.kv_len - u.q_len + u.row0 / G - p.window) : -1;
        v_norm = __uint_as_float((127u + 125u) << 23);  // no scale met yet: the largest power of two
      }
      // the largest V scale of the stage's keys that some row sees, and this lane's smallest; every warp computes the same
      uint32_t tb = 0;
      float low = INFINITY;
#pragma unroll
      for (int i = 0; i < kBN / 32; ++i) {
        const int key = pos + lane + 32 * i;
        if (key < kv_end && key > lo_min) {
          const float v = vs_s[(key >> sb_shift) - e0];
          tb = max(tb, __float_as_uint(v));
          low = fminf(low, v);
        }
      }
      tb = __reduce_max_sync(0xffffffffu, tb);  // positive floats order as integers
      if (__uint_as_float(tb) * v_norm >= (float)(2 << kVBits)) {
        uint32_t e = tb >> 23;
        e = e < 8u ? 8u : e;
        v_norm = __uint_as_float((254u + kVBits - e) << 23);
      }
      const bool far = __any_sync(0xffffffffu, low * v_norm < kFar);
      const float f_scale = far ? 0.f : v_norm, f_plus = far ? kFarV : 0.f;
      if (!mbar_wait(bar_kv_empty(st), ((gi / NS) & 1) ^ 1, abort_flag, wait_ns)) break;
      // each token's factor on its logits; in the common kernel one per 8 tokens
      if (ctid < (coarse ? kBN / 8 : kBN)) {
        const int key = pos + (coarse ? ctid * 8 : ctid);
        reinterpret_cast<float*>(smem + C::OFF_KSCALE + st * (kBN * 4))[ctid] = key < kv_end ? ks_s[(key >> sb_shift) - e0] * to_log2 : 1.f;
      }
      if (far && ctid < kBN) {
        const int key = pos + ctid;
        reinterpret_cast<float*>(smem + C::OFF_VSCALE + st * (kBN * 4))[ctid] = key < kv_end && key > lo_min ? vs_s[(key >> sb_shift) - e0] : 0.f;
      }
      if (ctid == 0) {
        metas[st] = meta;
        vrefs[st] = far ? -v_norm : v_norm;
      }
      const uint8_t* raw = smem + C::OFF_RAW + rs * C::RAW_BYTES + ch * 16;
      uint8_t* out = smem + C::OFF_KV + st * C::STAGE_BYTES + (ch >> 2) * 1024;
      // a short loop on purpose: the roles of this kernel share an instruction cache that their unrolled bodies overflow
#pragma unroll 1
      for (int t = t0; t < kBN; t += TSTEP) {
        const uint4 kc = *reinterpret_cast<const uint4*>(raw + t * D);
        uint4 vc = *reinterpret_cast<const uint4*>(raw + (kBN + t) * D);
        const int key = pos + t;
        float f = fmaf(vs_s[(key >> sb_shift) - e0], f_scale, f_plus);
        if (key >= kv_end || key <= lo_min) {  // V of a key that no row sees is zero: those are stale bytes, possibly NaN
          vc = make_uint4(0u, 0u, 0u, 0u);
          f = 0.f;
        }
        uint8_t* row = out + (uint32_t)(t >> 3) * C::GROUP_BYTES + (uint32_t)(t & 7) * 128;
        uint8_t* at0 = row + ((c_first ^ (uint32_t)(t & 7)) << 4);
        uint8_t* at1 = row + ((c_second ^ (uint32_t)(t & 7)) << 4);
        const uint32_t k0 = half_first ? kc.z : kc.x, k1 = half_first ? kc.w : kc.y, k2 = half_first ? kc.x : kc.z, k3 = half_first ? kc.y : kc.w;
        uint32_t w[4];
        Code::widen(k0, w[0], w[1]);
        Code::widen(k1, w[2], w[3]);
        *reinterpret_cast<uint4*>(at0) = make_uint4(w[0], w[1], w[2], w[3]);
        Code::widen(k2, w[0], w[1]);
        Code::widen(k3, w[2], w[3]);
        *reinterpret_cast<uint4*>(at1) = make_uint4(w[0], w[1], w[2], w[3]);
        const __half2 f2 = __float2half2_rn(f);
        const uint32_t v0 = half_first ? vc.z : vc.x, v1 = half_first ? vc.w : vc.y, v2 = half_first ? vc.x : vc.z, v3 = half_first ? vc.y : vc.w;
        Code::widen(v0, w[0], w[1]);
        Code::widen(v1, w[2], w[3]);
        *reinterpret_cast<uint4*>(at0 + C::V_OFF) = make_uint4(mul_f16x2(w[0], f2), mul_f16x2(w[1], f2), mul_f16x2(w[2], f2), mul_f16x2(w[3], f2));
        Code::widen(v2, w[0], w[1]);
        Code::widen(v3, w[2], w[3]);
        *reinterpret_cast<uint4*>(at1 + C::V_OFF) = make_uint4(mul_f16x2(w[0], f2), mul_f16x2(w[1], f2), mul_f16x2(w[2], f2), mul_f16x2(w[3], f2));
      }
      fence_async_smem();  // the MMAs read the stage through the async proxy
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_kv_full(st));
        mbar_arrive(bar_raw_empty(rs));
      }
      ++gi;
    }
  } else {
    take_registers<C::REGS_SOFTMAX>();
    // =============================== softmax warps ===============================
    // One thread per tile row: warp (x, quarter) owns rows quarter*32.. of tile x (the TMEM lanes a
    // warp may touch are fixed by warp % 4), so row maxima and sums need no shuffles.
    constexpr int HB = kBN;
    const int sw = warp - 8;
    const int x = sw / C::SM_WARPS;                       // which tile of the CTA
    const int row = (warp & 3) * 32 + lane;               // TMEM lane == row within the tile
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem_base + lane_addr + C::TMEM_S + x * kBN;
    const uint32_t tm_p0 = tmem_base + lane_addr + C::TMEM_P + x * 2 * C::P_COLS;
    const uint32_t tm_o = tmem_base + lane_addr + C::TMEM_O + x * D;
    int gi = 0;   // KV stage counter (all roles see the same stage sequence)
    int ti = 0;   // stages this tile took part in
    int k = 0;    // item counter (all roles see the same item sequence)
    bool alive = true;
    // The query row of an item goes to shared memory as f16 (K-major, 128B swizzle); a bf16 row by a power of two that takes
    // its largest element to [2^14, 2^15): exact for every element above 2^-28 of it, absolute error 2^-39 of it below.  The
    // row of the NEXT item is fetched under the last stage of the current one: the tile's query buffer is free as soon as
    // the item's last S has completed, and with the row in place the S issuer starts the next item while this thread is
    // still in the epilogue.
    uint8_t* q_row = smem + C::OFF_Q + x * C::Q_BYTES + (uint32_t)row * 128;
    float q_fac = 1.f, q_fac_next = 1.f;  // 2^-k of the row
    auto q_fetch = [&](const Unit& uu, int hh) {
      const int R = uu.row0 + x * kBM + row;
      const bool ok = R < uu.q_len * G;
      const int qt = R / G, g = R - qt * G;
      const uint4* src = reinterpret_cast<const uint4*>(p.q);
      if (ok) src += ((size_t)(uu.q_start + qt) * p.Hq + hh * G + g) * (D / 8);
      int e = 127 + 14;
      if constexpr (!std::is_same<T, __half>::value) {
        uint32_t big = 0;
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          const uint4 v = ok ? __ldg(src + c) : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) big = max(big, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
        }
        e = (int)(big >> 23);  // biased exponent of the row's largest element
        e = e == 255 ? 127 + 14 : (e < 20 ? 20 : e);  // infinities and NaN stay what they are; 2^k stays finite
      }
      const float up = __uint_as_float((uint32_t)(254 + 14 - e) << 23);
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {  // rows past the item's end are zero
        uint4 v = ok ? __ldg(src + c) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (!std::is_same<T, __half>::value) {
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = Mma<__half>::pack(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(q_row + (uint32_t)(c >> 3) * (kBM * 128) + (uint32_t)(((c & 7) ^ (row & 7)) << 4)) = v;
      }
      q_fac_next = __uint_as_float((uint32_t)(e - 14) << 23);
      fence_async_smem();  // the MMA reads the tile through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q_full(x));
    };
    bool q_ready = false;    // this item's query row was fetched during the previous item
    // The group follows the item sequence through the producer's item ring (a counter says how many
    // items have been published; an mbarrier parity could alias, because a group whose tile is idle
    // skips whole items) and counts stages itself, so that per stage it waits only for S.
    while (alive) {
      {
        bool have = *items_pub > k;
        if (!have) {
          const unsigned long long t0 = global_timer_ns();
          while (true) {
            __nanosleep(64);
            if (*items_pub > k) {
              have = true;
              break;
            }
            if (*abort_flag || global_timer_ns() - t0 > wait_ns) break;
          }
        }
        have = __all_sync(0xffffffffu, have);
        if (!have) {
          *abort_flag = 1;
          break;
        }
        __threadfence_block();  // the ring entry was written before the counter moved; read it after
      }
      const Unit u = ring[k % kRingP].u;
      const int h = ring[k % kRingP].h;
      const int first_stage = ring[k % kRingP].first_stage, quota = ring[k % kRingP].quota;
      ++k;
      if (u.seq < 0) break;
      int n_stages = (u.kv_end - u.kv_begin + kBN - 1) / kBN;
      if (n_stages < 1) n_stages = 1;
      const bool two = u.slot > kBM && u.q_len * G > u.row0 + kBM;  // the item has rows for both tiles
      const bool active = (x == 0) || two;
      if (!active) {  // the item has no rows for this tile
        __syncwarp();
        if (lane == 0) {
          __threadfence_block();  // the ring entry has been read
          atomicAdd(const_cast<int*>(&skipped[x]), 1);
        }
        gi += n_stages;
        continue;
      }
      // ---- new item: row bookkeeping and the query row (K-major, 128B swizzle) ----
      const int rows_total = u.q_len * G;
      const int R = u.row0 + x * kBM + row;
      const bool row_ok = R < rows_total;
      const int qt = R / G, g = R - qt * G;
      const int out_row_q = u.q_start + qt;
      const int out_head = h * G + g;
      const int pos_row = row_ok ? (u.kv_len - u.q_len + qt) : -1;
      const int lo_row = (p.window > 0) ? pos_row - p.window : -1;
      float m_run = -INFINITY, l_run = 0.f, v_norm = 0.f;
      if (!q_ready) {
        // all S MMAs of this tile's previous item completed before its last s_full fired, which
        // this thread waited for, so the query tile may be overwritten
        q_fetch(u, h);
      }
      q_ready = false;
      q_fac = q_fac_next;
      // runs of common stages, and the far ones between them
      int js = 0;
      while (true) {
        bool far = false;
        for (; js < n_stages; ++js, ++gi, ++ti) {
          const int st = gi % NS;
          const int pos = u.kv_begin + js * kBN;  // first key of the stage
          const bool first = (js == 0);
          if (!mbar_wait(bar_s_full(x), ti & 1, abort_flag, wait_ns)) { alive = false; break; }
          tc_fence_after();
          // ---- the row's logits of the stage into registers; then the S columns are free for the
          // tile's next S MMA, which runs while this stage's exponentials are computed
          uint32_t sr[HB];
#pragma unroll
          for (int c = 0; c + 32 <= HB; c += 32) tc_ld32(tm_s + c, *reinterpret_cast<uint32_t(*)[32]>(&sr[c]));
          static_assert(HB % 32 == 0, "S is read 32 columns at a time");
          const float v_stage = vrefs[st];  // on its way with S
          const float4* kf4 = reinterpret_cast<const float4*>(smem + C::OFF_KSCALE + st * (kBN * 4));
          tc_wait_ld();
          if (__builtin_expect(v_stage < 0.f, 0)) {
            far = true;
            break;
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_s_free(x));

          // ---- logits in the log2 domain: raw dot products times the token's factor (k_scale * scale * log2 e) and the row's.
          // Common case: the products stay in the registers, a factor per 8 columns goes into the exponent's FMA and only the
          // groups' maxima are multiplied; a soft cap, finer scales or a scale that is not positive materialise the logits.
          const bool full_vis = (pos + HB - 1 <= pos_row) && (pos > lo_row);
          float ef[HB / 8];
#pragma unroll
          for (int i = 0; i < HB / 8; ++i) ef[i] = 1.f;
          if constexpr (PLAIN) {
#pragma unroll
            for (int i = 0; i < HB / 8; i += 4) {
              const float4 f = kf4[i >> 2];
              // not below the smallest normal number: a masked logit, -inf, times 0 would be NaN
              ef[i] = fmaxf(f.x * q_fac, 1.17549435e-38f);
              ef[i + 1] = fmaxf(f.y * q_fac, 1.17549435e-38f);
              ef[i + 2] = fmaxf(f.z * q_fac, 1.17549435e-38f);
              ef[i + 3] = fmaxf(f.w * q_fac, 1.17549435e-38f);
            }
          }
          if constexpr (!PLAIN) {
            const uint64_t qf = pack_f32x2(q_fac, q_fac);
#pragma unroll
            for (int i = 0; i < HB; i += 4) {
              const float4 f = kf4[i >> 2];
              const float2 a = unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), mul_f32x2(pack_f32x2(f.x, f.y), qf)));
              const float2 b = unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3])), mul_f32x2(pack_f32x2(f.z, f.w), qf)));
              sr[i] = __float_as_uint(a.x);
              sr[i + 1] = __float_as_uint(a.y);
              sr[i + 2] = __float_as_uint(b.x);
              sr[i + 3] = __float_as_uint(b.y);
            }
            if (p.cap != 0.f) {
              // cap * tanh(t) = cap - 2 cap / (2^(2 t log2 e) + 1); the factors hold the 2 log2 e.  An infinite power gives cap
              const uint64_t one = pack_f32x2(1.f, 1.f), cap = pack_f32x2(p.cap_log2, p.cap_log2), twice = pack_f32x2(-2.f * p.cap_log2, -2.f * p.cap_log2);
#pragma unroll
              for (int i = 0; i < HB; i += 2) {
                const float2 e = unpack_f32x2(add_f32x2(pack_f32x2(fast_exp2(__uint_as_float(sr[i])), fast_exp2(__uint_as_float(sr[i + 1]))), one));
                const float2 y = unpack_f32x2(fma_f32x2(pack_f32x2(fast_reciprocal(e.x), fast_reciprocal(e.y)), twice, cap));
                sr[i] = __float_as_uint(y.x);
                sr[i + 1] = __float_as_uint(y.y);
              }
            }
          }
          if (__builtin_expect(!full_vis, 0)) {
            const int hi_i = pos_row - pos;  // last visible column of the stage
            const int lo_i = lo_row - pos;   // columns up to here are left of the window
#pragma unroll
            for (int i = 0; i < HB; ++i)
              if (i > hi_i || i <= lo_i) sr[i] = __float_as_uint(-INFINITY);
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < HB; i += 8) {
            float a = fmaxf(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
            float b = fmaxf(__uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3]));
            a = fmax3(a, __uint_as_float(sr[i + 4]), __uint_as_float(sr[i + 5]));
            b = fmax3(b, __uint_as_float(sr[i + 6]), __uint_as_float(sr[i + 7]));
            mx = fmaxf(mx, fmaxf(a, b) * ef[i >> 3]);
          }
          // P_x has two buffers: this stage's goes where the stage before the previous one's was, whose
          // P.V must have read it (it has, normally long ago)
          if (ti >= 2) {
            if (!mbar_wait(bar_pv_done(x, ti & 1), ((ti - 2) >> 1) & 1, abort_flag, wait_ns)) { alive = false; break; }
          }
          const uint32_t tm_p = tm_p0 + (ti & 1) * C::P_COLS;
          // O comes into the stage's units if the row sees a key of it; they never grow finer over an item
          const float v_new = mx > -INFINITY ? v_stage : v_norm;
          // the row's maximum has outgrown its reference, or V comes in other units than O's
          const bool grow = (mx > m_run + kLazyP) || (m_run == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xffffffffu, grow || v_new != v_norm)) {
            float alpha = 1.f;
            if (m_run > -INFINITY) alpha = v_new * power_of_two_inverse(v_norm);  // O is zero otherwise
            if (grow) {
              const float f = fast_exp2(m_run - (mx - kRefBelow));  // 0 on the first finite maximum
              m_run = mx - kRefBelow;
              l_run *= f;
              alpha *= f;
            }
            v_norm = v_new;
            if (!first) {
              // O holds the sum over the earlier stages of this item: rescale the row, once the tile's
              // previous P.V has completed (O is only touched between P.Vs)
              if (!mbar_wait(bar_pv_done(x, (ti - 1) & 1), ((ti - 1) >> 1) & 1, abort_flag, wait_ns)) { alive = false; break; }
              tc_fence_after();
#pragma unroll 1
              for (int c0 = 0; c0 < D; c0 += 16) {
                uint32_t o[16];
                tc_ld16(tm_o + c0, o);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                tc_st16(tm_o + c0, o);
              }
            }
          }
          const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
          // probabilities, packed as 16-bit pairs, into the tile's P buffer of this stage
          // (pairs of columns in one instruction where there is one: this loop's length bounds the kernel)
          const uint64_t neg_m = pack_f32x2(-m_use, -m_use);
          uint64_t lsum[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < HB; c += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float f = ef[(c + 2 * j) >> 3];
              const uint64_t y = fma_f32x2(pack_f32x2(__uint_as_float(sr[c + 2 * j]), __uint_as_float(sr[c + 2 * j + 1])), pack_f32x2(f, f), neg_m);
              const float2 e = unpack_f32x2(y);
              const float p0 = fast_exp2(e.x), p1 = fast_exp2(e.y);
              lsum[j & 1] = add_f32x2(lsum[j & 1], pack_f32x2(p0, p1));
              pk[j] = Mma<__half>::pack(p0, p1);
            }
            tc_st16(tm_p + (c >> 1), pk);
          }
          const float2 lsum_pair = unpack_f32x2(add_f32x2(lsum[0], lsum[1]));
          l_run += lsum_pair.x + lsum_pair.y;
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p_full(x, ti & 1));
        }
        if (!far) break;
        const int st = gi % NS;
        const FarRow r = far_stage<D, PLAIN>(
            {m_run, l_run, v_norm, true}, reinterpret_cast<const float*>(smem + C::OFF_KSCALE + st * (kBN * 4)),
            reinterpret_cast<const float*>(smem + C::OFF_VSCALE + st * (kBN * 4)), q_fac, p.cap_log2, pos_row - (u.kv_begin + js * kBN),
            lo_row - (u.kv_begin + js * kBN), tm_s, tm_p0 + (ti & 1) * C::P_COLS, tm_o, bar_s_free(x), bar_p_full(x, ti & 1),
            bar_pv_done(x, ti & 1), bar_pv_done(x, (ti - 1) & 1), ti, js == 0, abort_flag, wait_ns);
        if (!r.ok) { alive = false; break; }
        m_run = r.m;
        l_run = r.l;
        v_norm = r.v;
        ++js, ++gi, ++ti;
      }
      if (!alive) break;
      // ---- last stage of the piece.  All S of the item completed long ago, so the tile's query buffer is free: fetch
      // the next item's query row (if the producer has published that item already; it normally has, it runs stages
      // ahead), then wait for the last P.V, normalise and store, or (a part of a split item) publish the unnormalised
      // part and, if it is the last to arrive, combine ----
      bool q_pending = *items_pub > k;
      q_pending = __all_sync(0xffffffffu, q_pending);
      if (q_pending) {
        __threadfence_block();
        const Unit un = ring[k % kRingP].u;
        q_pending = un.seq >= 0 && (x == 0 || (un.slot > kBM && un.q_len * G > un.row0 + kBM));
        if (q_pending) {
          q_fetch(un, ring[k % kRingP].h);
          q_ready = true;
        }
      }
      if (!mbar_wait(bar_pv_done(x, (ti - 1) & 1), ((ti - 1) >> 1) & 1, abort_flag, wait_ns)) { alive = false; break; }
      tc_fence_after();
      const float v_back = power_of_two_inverse(v_norm);  // O is in units of v_ref
      if (u.n_chunks > 1) {
        // Slot of the part CTA c holds of this (item, head): a CTA has at most two parts, the item
        // its quota begins in (slot 2c) and the item its quota ends in (slot 2c + 1).
        auto slot_of = [&](int c) { return ((long long)first_stage <= (long long)c * quota) ? 2 * c : 2 * c + 1; };
        const size_t mine = ((size_t)slot_of((int)blockIdx.x) * NT + x) * kBM + row;
        if (row_ok) p.ppart_ml[mine] = make_float2(m_run, l_run);
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          tc_ld32(tm_o + c0, o);
          tc_wait_ld();
          if (row_ok) {
            float4* dst = reinterpret_cast<float4*>(p.ppart_o + mine * D + c0);
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              dst[c >> 2] = make_float4(__uint_as_float(o[c]) * v_back, __uint_as_float(o[c + 1]) * v_back,
                                        __uint_as_float(o[c + 2]) * v_back, __uint_as_float(o[c + 3]) * v_back);
          }
        }
        tc_fence_before();
        __threadfence();
        __syncwarp();
        int old = 0;
        if (lane == 0) {
          mbar_arrive(bar_o_free(x));
          // one counter per 32-row quarter of the tile: the warps of a group never wait for each other
          old = atomicAdd(&p.ptickets[((size_t)u.merge_idx * NT + x) * 4 + (warp & 3)], 1);
        }
        old = __shfl_sync(0xffffffffu, old, 0);
        if (old == u.n_chunks - 1 && row_ok) {
          // last part to arrive: combine the parts of this row, in part order (so the result does not
          // depend on which part arrived last)
          __threadfence();
          const int c_first = first_stage / quota;
          float m_tot = -INFINITY;
          for (int pi = 0; pi < u.n_chunks; ++pi)
            m_tot = fmaxf(m_tot, __ldcg(&p.ppart_ml[((size_t)slot_of(c_first + pi) * NT + x) * kBM + row]).x);
          const float mu = (m_tot == -INFINITY) ? 0.f : m_tot;
          float l_tot = 0.f;
          for (int pi = 0; pi < u.n_chunks; ++pi) {
            const float2 ml = __ldcg(&p.ppart_ml[((size_t)slot_of(c_first + pi) * NT + x) * kBM + row]);
            l_tot += ml.y * fast_exp2(ml.x - mu);
          }
          float scl = 1.f, l_fin = l_tot;
          if (p.num_sinks > 0) {
            const int srow = (p.sink_rows == p.Hq) ? out_head : (p.sink_rows == Hkv ? h : 0);
            const float* sk = p.sinks + (size_t)srow * p.num_sinks;
            float sm = -INFINITY;
            for (int i = 0; i < p.num_sinks; ++i) sm = fmaxf(sm, sk[i] * kLog2eP);
            const float m_fin = fmaxf(m_tot, sm);
            const float mf = (m_fin == -INFINITY) ? 0.f : m_fin;
            scl = fast_exp2(m_tot - mf);
            l_fin = l_tot * scl;
            for (int i = 0; i < p.num_sinks; ++i) l_fin += fast_exp2(sk[i] * kLog2eP - mf);
          }
          scl = (l_fin > 0.f) ? scl / l_fin : 0.f;
          T* orow = reinterpret_cast<T*>(p.out) + ((size_t)out_row_q * p.Hq + out_head) * D;
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 32) {
            float acc[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[c] = 0.f;
            for (int pi = 0; pi < u.n_chunks; ++pi) {
              const size_t at = ((size_t)slot_of(c_first + pi) * NT + x) * kBM + row;
              const float f = fast_exp2(__ldcg(&p.ppart_ml[at]).x - mu);
              const float4* src = reinterpret_cast<const float4*>(p.ppart_o + at * D + c0);
#pragma unroll
              for (int c = 0; c < 32; c += 4) {
                const float4 v = __ldcg(src + (c >> 2));
                acc[c] += v.x * f;
                acc[c + 1] += v.y * f;
                acc[c + 2] += v.z * f;
                acc[c + 3] += v.w * f;
              }
            }
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
              uint4 v;
              v.x = Mma<T>::pack(acc[c] * scl, acc[c + 1] * scl);
              v.y = Mma<T>::pack(acc[c + 2] * scl, acc[c + 3] * scl);
              v.z = Mma<T>::pack(acc[c + 4] * scl, acc[c + 5] * scl);
              v.w = Mma<T>::pack(acc[c + 6] * scl, acc[c + 7] * scl);
              *reinterpret_cast<uint4*>(orow + c0 + c) = v;
            }
          }
        }
        continue;  // on to the next piece
      }
      const float l_row = l_run;
      float scl = 1.f, l_fin = l_row;
      if (p.num_sinks > 0 && row_ok) {
        // attention sinks join the denominator only
        const int srow = (p.sink_rows == p.Hq) ? out_head : (p.sink_rows == Hkv ? h : 0);
        const float* sk = p.sinks + (size_t)srow * p.num_sinks;
        float sm = -INFINITY;
        for (int i = 0; i < p.num_sinks; ++i) sm = fmaxf(sm, sk[i] * kLog2eP);
        const float m_fin = fmaxf(m_run, sm);
        const float mf = (m_fin == -INFINITY) ? 0.f : m_fin;
        scl = fast_exp2(m_run - mf);
        l_fin = l_row * scl;
        for (int i = 0; i < p.num_sinks; ++i) l_fin += fast_exp2(sk[i] * kLog2eP - mf);
      }
      scl = (l_fin > 0.f) ? scl / l_fin : 0.f;
      // two factors: their product can lie below what float32 holds, where the scales are tiny and the keys many
      auto finish = [&](uint32_t o) { return __uint_as_float(o) * scl * v_back; };
      T* orow = reinterpret_cast<T*>(p.out) + ((size_t)out_row_q * p.Hq + out_head) * D;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        tc_ld32(tm_o + c0, o);
        tc_wait_ld();
        if (row_ok) {
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            uint4 v;
            v.x = Mma<T>::pack(finish(o[c]), finish(o[c + 1]));
            v.y = Mma<T>::pack(finish(o[c + 2]), finish(o[c + 3]));
            v.z = Mma<T>::pack(finish(o[c + 4]), finish(o[c + 5]));
            v.w = Mma<T>::pack(finish(o[c + 6]), finish(o[c + 7]));
            *reinterpret_cast<uint4*>(orow + c0 + c) = v;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_o_free(x));
    }
  }
  if (*abort_flag) flags |= EJK_RPA_ST_TIMEOUT;
  // every role has left its loop (all waits are bounded), so the TMEM can go back
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(C::TMEM_COLS) : "memory");
  }
  if (flags && p.status) atomicOr(reinterpret_cast<unsigned*>(p.status), flags);
}

template <typename T, typename Code, int D, bool PLAIN>
cudaError_t launch_one(const Params& p, const Q8Cache& c, int n_sm, cudaStream_t stream, bool pdl) {
  using C = CfgP<D>;
  auto kern = q8_prefill_kernel<T, Code, D, PLAIN>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return e;
    // a register split beyond what the block is launched with would wait forever: refuse it
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, kern);
    if (e != cudaSuccess) return e;
    if (at.numRegs < C::REGS) return cudaErrorInvalidConfiguration;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  return launch_kernel(kern, dim3(n_sm), dim3(C::THREADS), C::SMEM_BYTES, stream, pdl, p, c);
}

template <typename T, typename Code>
cudaError_t dispatch(const Params& p, const Q8Cache& c, int n_sm, cudaStream_t stream, bool pdl) {
  const bool plain = c.block_shift >= 3 && p.cap == 0.f && p.scale_log2 > 0.f;
  switch (p.D) {
    case 64: return plain ? launch_one<T, Code, 64, true>(p, c, n_sm, stream, pdl) : launch_one<T, Code, 64, false>(p, c, n_sm, stream, pdl);
    case 128: return plain ? launch_one<T, Code, 128, true>(p, c, n_sm, stream, pdl) : launch_one<T, Code, 128, false>(p, c, n_sm, stream, pdl);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

bool q8_prefill_supported(int head_dim) { return head_dim == 64 || head_dim == 128; }

cudaError_t launch_q8_prefill(const Params& p, const Q8Cache& c, int dtype, int code, int n_sm, cudaStream_t stream, bool pdl) {
  if (code == EJK_Q8_I8)
    return dtype == EJK_RPA_BF16 ? dispatch<__nv_bfloat16, CodeI8>(p, c, n_sm, stream, pdl) : dispatch<__half, CodeI8>(p, c, n_sm, stream, pdl);
  return dtype == EJK_RPA_BF16 ? dispatch<__nv_bfloat16, CodeE4M3>(p, c, n_sm, stream, pdl) : dispatch<__half, CodeE4M3>(p, c, n_sm, stream, pdl);
}

}  // namespace ejk
