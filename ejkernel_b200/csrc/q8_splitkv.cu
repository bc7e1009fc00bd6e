// Split-KV ragged attention over the 8-bit cache: decode rows and short chunks.
//
//   x_j  = scale * k_scale_j * (q . k_j),  p_j = 2^(x_j log2 e - m)   (m: running maximum, lazily moved)
//   O   += (p_j * v_scale_j) v_j,  l += p_j;   out = O / l
//
// The kernel is a stream of the cache: every byte of K and V is read once per kv head and costs 2 * G multiply-adds, so
// DRAM bounds it, and everything else has to stay out of the way.
//   * Work: the 128-token stages of all (row tile, kv head) pairs form one sequence that is cut into equal quotas, one per
//     CTA.  Every CTA finds its quota itself, from the lengths (a scan that all CTAs do at the same time: of a microsecond for decode
//     rows, but one thread walks all row tiles of a sequence, one after the other, which a long prompt at head_dim 256 feels):
//     no planner runs before this kernel, no queue is drawn from, no SM waits for the last item of another.  A pair that
//     straddles a quota boundary is finished by several CTAs; the last of them to arrive combines their parts, in part order,
//     sixteen at a time.  A CTA has two partial pieces at most, so the parts of all calls fit 2 slots per CTA.
//   * A stage is 128 tokens of one head, fetched by one producer warp as TMA boxes of up to 64 tokens.  A head's page is
//     contiguous, so a box of 16 tokens at head_dim 128 is two runs of 2 KB.  A second producer warp brings what goes with the
//     stage: its scales, with 4-byte cp.async copies that arrive on the same mbarrier, and the query rows of a new piece.  (With
//     one warp for both, its latency per stage, 1.4 us, bounded the kernel.)
//   * Four consumer warps take 32 tokens each.  Codes go to f16 in registers, which is exact for both types, and both
//     products run on f16 mma.sync with float32 sums.  8-bit operands would halve the mma work, which is not what bounds
//     the kernel, and would round q and p to 3 bits of mantissa.  (Eight warps in two teams that take the stages in turn
//     were slower: 0.50 ms against 0.37 for 128 sequences of 8192 keys; the registers go down to 96.)
//   * k_scale multiplies the finished dot product, v_scale the probability: two multiplications a token and row, none per
//     element.  p * v_scale has to fit f16: a warp divides v_scale by a power of two, chosen from the largest scale that
//     it has met so that the product is at most 2^15, and moves it as it moves m.  What is below 2^-24 of that range is lost:
//     2^-31 of the largest |V| that the row sees.  In a tile of several tokens the largest scale met can be one that the mask hides
//     from a row; where scales lie 2^11 and more apart there, the piece's rows are computed one by one at its end (far_row).
//   * bf16 queries go to f16 by a power of two per row (their largest element to [2^14, 2^15)), undone on the logits.
//
// Every wait on an mbarrier is bounded in wall time (option "wait_ms"): on expiry the warp raises
// EJK_RPA_ST_TIMEOUT, sets the CTA's abort flag and returns, and every other wait of the CTA gives up as soon as it sees it.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr int kConsumerWarps = 4;
constexpr int kThreads = (kConsumerWarps + 2) * 32;
constexpr int kRing = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMergeInFlight = 8;     // parts whose loads a merge keeps in flight per row
constexpr int kGroup = 16;            // parts that are combined at a time: more go through groups
constexpr float kLazyRescale = 8.0f;  // rescale the accumulators only when the max grows by 2^8: p <= 2^8
constexpr float kFar = 0x1p-5f;       // a scale below this in those units lies far from the largest: see far_row
constexpr int kVBits = 6;             // the largest v_scale met so far is taken to [2^6, 2^7): p * v_scale <= 2^15 < 65504

// One piece of work of a CTA: stages of one (row tile, kv head).  Of a pair that several CTAs share, u.n_chunks is the number of
// parts, u.chunk_idx this part's number and u.merge_idx the CTA of part 0; u.slot is where this part goes, u.pad where part 0 is.
struct ItemDesc {
  Unit u;
  int32_t h;
  int32_t first;  // the CTA's first piece
  int32_t pad[2];
};

// What a CTA works out before it starts: the sequences that hold the first and the last stage of its quota, and the stages (per
// head) of the sequences before them.
struct Share {
  long long base[2];
  int seq[2];
};

template <int D, int NT, int NS>
struct Cfg {
  static constexpr int TK = 128;                  // tokens per stage
  static constexpr int TW = TK / kConsumerWarps;  // tokens of a stage per consumer warp
  static constexpr int RB = D < 128 ? D : 128;    // bytes of a row in one swizzled column (the swizzle span)
  static constexpr int DC = D / RB;               // columns
  static constexpr int CH = RB / 16;              // 16-byte chunks of a column's row
  static constexpr int RT = 8 * NT;
  static constexpr int STAGE_BYTES = TK * 2 * D;
  static constexpr int Q_ROW_BYTES = D * 2 + 16;
  static constexpr int Q_BYTES = RT * Q_ROW_BYTES;
  static constexpr int OFF_SCALE = NS * STAGE_BYTES;              // per stage: TK scales of K, TK of V (at most)
  static constexpr int OFF_Q = OFF_SCALE + NS * 2 * TK * 4;
  static constexpr int OFF_QFAC = OFF_Q + NS * Q_BYTES;           // per stage: 2^-k of each query row
  static constexpr int OFF_ML = (OFF_QFAC + NS * RT * 4 + 7) / 8 * 8;  // two pieces' (m, l) of each warp and row
  static constexpr int OFF_RING = (OFF_ML + 2 * kConsumerWarps * RT * 8 + 63) / 64 * 64;
  static constexpr int OFF_META = OFF_RING + kRing * (int)sizeof(ItemDesc);
  static constexpr int OFF_BAR = OFF_META + NS * 8;  // full[NS], empty[NS], cbar
  static constexpr int OFF_SHARE = OFF_BAR + (2 * NS + 1) * 8;
  static constexpr int OFF_ABORT = OFF_SHARE + (int)sizeof(Share);
  static constexpr int OFF_BAD = OFF_ABORT + 4;
  static constexpr int SMEM_BYTES = OFF_ABORT + 16 + 1024;  // + alignment slack
  static constexpr int CTAS = SMEM_BYTES <= 112 * 1024 ? 2 : 1;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
  static_assert(kConsumerWarps * RT * D * 4 <= STAGE_BYTES, "a piece's last stage takes the warps' accumulators");
  static_assert(NT == 2 || D == 256 || CTAS == 2, "two CTAs per SM for the usual shapes");
};

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
// 4-byte asynchronous copy, and the arrival that follows this thread's copies (counted in the barrier's expected count)
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// ---- the stages of a sequence ----
struct Seq {
  int q_start, q_len, kv_len, tiles;  // tiles = 0: nothing to do here
};
__device__ __forceinline__ Seq load_seq(const Params& p, int s, int rows_per_tile, unsigned& flags) {
  const int q0 = __ldg(p.query_start_loc + s), q1 = __ldg(p.query_start_loc + s + 1);
  int kv = __ldg(p.context_lens + s);
  const int kv_cap = p.pages_per_seq * p.page_size;
  if (kv < 0 || kv > kv_cap) {
    flags |= EJK_RPA_ST_KVLEN;
    kv = kv < 0 ? 0 : kv_cap;
  }
  int ql = q1 - q0;
  if (bad_rows(q0, q1, p.T)) {
    flags |= EJK_RPA_ST_QLEN;
    ql = 0;
  }
  if (ql > kv) flags |= EJK_RPA_ST_QLEN;  // rows at negative positions see no key and produce 0
  const int rows = ql * p.G;
  const bool tiles_elsewhere = p.prefill_min_rows > 0 && rows >= p.prefill_min_rows;  // served by tensor tiles
  return {q0, ql, kv, tiles_elsewhere ? 0 : (rows + rows_per_tile - 1) / rows_per_tile};
}
// keys [lo, hi) that some row of tile t sees; lo is rounded down to where boxes may start.  Returns the stages, at least one
__device__ __forceinline__ int tile_stages(const Params& p, const Seq& q, int t, int rows_per_tile, int& lo, int& hi) {
  const int r_first = t * rows_per_tile;
  const int r_last = min(r_first + rows_per_tile, q.q_len * p.G) - 1;
  const int base = q.kv_len - q.q_len;
  hi = max(base + r_last / p.G + 1, 0);
  lo = 0;
  if (p.window > 0) lo = max(base + r_first / p.G - p.window + 1, 0) / kTileTokens * kTileTokens;
  hi = max(hi, lo);
  return max((hi - lo + 127) >> 7, 1);
}
__device__ __forceinline__ long long seq_stages(const Params& p, const Seq& q, int rows_per_tile) {
  long long n = 0;
  int lo, hi;
  for (int t = 0; t < q.tiles; ++t) n += tile_stages(p, q, t, rows_per_tile, lo, hi);
  return n;
}

// ---- combining the parts of a pair ----
// Arrival counters, three per CTA and consumer warp (each merges rows of its own), zero between calls: atomicInc with the number of arrivals as its limit takes a counter back to
// zero with the last of them.  [c]: the first sixteen parts of the pair that begins in CTA c; [n + c]: the sixteen parts that
// begin with CTA c's, of a pair that begins earlier; [2n + c]: the groups of the pair that begins in CTA c.
struct Arrival {
  int count;   // parts (or groups) to combine now; 0: others are still to come
  int stride;  // in parts
  int part0;
  bool last;   // they are all there is
};
__device__ __forceinline__ Arrival arrive_part(int* tickets, int n_cta, int c0, int part, int n_parts) {
  const int g = part / kGroup;
  const int size = min(kGroup, n_parts - g * kGroup);
  const unsigned old = atomicInc(reinterpret_cast<unsigned*>(tickets + (g ? n_cta + c0 + g * kGroup : c0)), (unsigned)size - 1u);
  return {old == (unsigned)size - 1u ? size : 0, 1, g * kGroup, n_parts <= kGroup};
}
__device__ __forceinline__ Arrival arrive_group(int* tickets, int n_cta, int c0, int n_parts) {
  const int groups = (n_parts + kGroup - 1) / kGroup;
  const unsigned old = atomicInc(reinterpret_cast<unsigned*>(tickets + 2 * n_cta + c0), (unsigned)groups - 1u);
  return {old == (unsigned)groups - 1u ? groups : 0, kGroup, 0, true};
}

// The power of two that takes the largest V scale met to [2^6, 2^7)
__device__ __forceinline__ float scale_unit(float top) {
  uint32_t e = __float_as_uint(top) >> 23;
  e = e < 8u ? 8u : e;
  return __uint_as_float((254u + kVBits - e) << 23);
}

// One query row of a piece by one warp, everything in float32: a lane computes one key's logit, then the lanes share out head_dim.
// It is for tiles of several tokens where a scale of V that some row does not see lies far above one that it does: one power of
// two for the tile's rows would push what the latter multiplies out of f16.  A call, at the end of the piece: the code of such
// cases in line cost decode batches 2 to 7 % and prompts at head_dim 256 up to 20 %.  Slow where it is taken, which data of one model
// is not expected to do: 64 requests of 4 tokens over 4096 keys 9.0 ms with scales 2^-40 to 1 at random, 0.22 ms without.
struct FarRow {
  const void* q;
  const int32_t* table;
  const uint8_t* pages;
  const float* scales;
  int32_t num_pages, page_size, Hkv, h, block_shift, key0, key1;
  float scale_log2, cap_log2, inv_cap_scale;  // cap_log2 == 0: no cap
  float m, l, o[8];                           // out: maximum, sum, this lane's columns
};
template <typename T, typename Code, int D>
__device__ __noinline__ void far_row(FarRow* r) {
  constexpr int VPL = D / 32;
  const int lane = threadIdx.x & 31, bpp = r->page_size >> r->block_shift;
  const T* q = static_cast<const T*>(r->q);
  float m = -INFINITY, l = 0.f, o[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) o[i] = 0.f;
#pragma unroll 1
  for (int base = r->key0; base < r->key1; base += 32) {
    const int key = base + lane;
    float y = -INFINITY, vs = 0.f;
    long long v_row = 0;
    if (key < r->key1) {
      const int pi = key / r->page_size, off = key - pi * r->page_size;
      int page = r->table[pi];
      if ((unsigned)page >= (unsigned)r->num_pages) page = 0;  // reported by the producer
      const long long plane = ((long long)page * r->Hkv + r->h) * 2;
      const uint8_t* k = r->pages + (plane * r->page_size + off) * D;
      const float ks = r->scales[plane * bpp + (off >> r->block_shift)];
      vs = r->scales[(plane + 1) * bpp + (off >> r->block_shift)];
      v_row = ((plane + 1) * r->page_size + off) * D;
      float dot = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; d += 16) {
        const uint4 c = *reinterpret_cast<const uint4*>(k + d);
        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf(Code::decode((uint8_t)(cw[i >> 2] >> (8 * (i & 3)))), to_float(q[d + i]), dot);
      }
      dot *= ks;
      y = r->cap_log2 != 0.f ? r->cap_log2 * soft_cap_tanh(dot * r->inv_cap_scale) : dot * r->scale_log2;
    }
    float top = y;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float m_new = fmaxf(m, top), mu = m_new == -INFINITY ? 0.f : m_new;
    const float f = fast_exp2(m - mu), e = fast_exp2(y - mu);
    m = m_new;
    float sum = e;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    l = l * f + sum;
#pragma unroll
    for (int i = 0; i < VPL; ++i) o[i] *= f;
    const float w = key < r->key1 ? e * vs : 0.f;
    const int n = min(r->key1 - base, 32);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const uint8_t* v = r->pages + __shfl_sync(0xffffffffu, v_row, j) + lane * VPL;
#pragma unroll
      for (int i = 0; i < VPL; ++i) o[i] = fmaf(wj, Code::decode(v[i]), o[i]);
    }
  }
  r->m = m;
  r->l = l;
#pragma unroll
  for (int i = 0; i < VPL; ++i) r->o[i] = o[i];
}

template <typename T, typename Code, int D, int NT, int NS>
__global__ void __launch_bounds__(kThreads, (Cfg<D, NT, NS>::CTAS))
q8_splitkv_kernel(const __grid_constant__ CUtensorMap tmap, const Params p, const Q8Cache cache) {
  using C = Cfg<D, NT, NS>;
  constexpr int TK = C::TK, RT = C::RT, TW = C::TW, CH = C::CH;
  constexpr int KT = D / 16;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem_base = smem_u32(smem);
  float2* mlbuf = reinterpret_cast<float2*>(smem + C::OFF_ML);
  ItemDesc* ring = reinterpret_cast<ItemDesc*>(smem + C::OFF_RING);
  int2* metas = reinterpret_cast<int2*>(smem + C::OFF_META);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_ABORT);
  volatile int* bad_offsets = reinterpret_cast<volatile int*>(smem + C::OFF_BAD);
  Share* share = reinterpret_cast<Share*>(smem + C::OFF_SHARE);
  const uint32_t bar_full = smem_base + C::OFF_BAR;
  const uint32_t bar_empty = bar_full + NS * 8;
  const uint32_t bar_c = bar_empty + NS * 8;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int Hkv = p.Hkv, G = p.G;
  const int pb = p.tma_block_tokens;  // tokens per TMA box (power of two, 8 to 64)
  const int pb_shift = p.tma_block_shift;
  const int sb_shift = cache.block_shift;
  const unsigned long long wait_ns = (unsigned long long)p.wait_timeout_ms * 1000000ull;
  unsigned flags = 0;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(bar_full + s * 8, 2 + 32);  // both producers' announcements, and every scale copying lane
      mbar_init(bar_empty + s * 8, kConsumerWarps);
    }
    mbar_init(bar_c, kConsumerWarps);
    *abort_flag = 0;
    *bad_offsets = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  __syncthreads();
  // launched as a programmatic dependent: everything above overlapped the tail of what came before.  Behind the tensor-tile
  // kernel there is nothing to wait for: it is released by CTAs that have themselves waited for all earlier work
  if (p.pdl & 2) pdl_wait();

  // ---- this CTA's quota of the stages
  int S = __ldg(p.num_seqs);
  if (S > p.S_max) {
    flags |= EJK_RPA_ST_NUM_SEQS;
    S = p.S_max;
  }
  if (S < 0) S = 0;
  const int n_cta = (int)gridDim.x;
  int quota;
  long long g0, g1;
  {
    long long* s_sum = reinterpret_cast<long long*>(mlbuf);  // not in use yet
    const int per = (S + kThreads - 1) / kThreads;
    const int a = min(tid * per, S), b = min(a + per, S);
    long long mine = 0;
    for (int i = a; i < b; ++i) mine += seq_stages(p, load_seq(p, i, RT, flags), RT);
    if (flags & EJK_RPA_ST_QLEN) *bad_offsets = 1;
    if (blockIdx.x != 0) flags = 0;  // one CTA reports
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    long long before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w];
    }
    const long long all = total * Hkv;
    const long long even = (all + n_cta - 1) / n_cta;
    quota = (int)max(even, (long long)(p.min_chunk >> 7));  // shorter pieces cost more to combine than they save
    g0 = min((long long)blockIdx.x * quota, all);
    g1 = min(g0 + quota, all);
    if (g0 < g1 && mine > 0) {
      for (int e = 0; e < 2; ++e) {
        const long long g = e ? g1 - 1 : g0;
        if (g < before * Hkv || g >= (before + mine) * Hkv) continue;
        long long base = before;
        unsigned none = 0;
        for (int i = a; i < b; ++i) {
          const long long n = seq_stages(p, load_seq(p, i, RT, none), RT);
          if (g < (base + n) * Hkv) {
            share->base[e] = base;
            share->seq[e] = i;
            break;
          }
          base += n;
        }
      }
    }
    __syncthreads();
  }

  if (warp >= kConsumerWarps) {
    // =============================== producer warps ===============================
    // Both walk the same pieces and stages.  The first issues the stages' boxes; the second brings their scales and, with the
    // first stage of a piece, its descriptor and query rows.
    const bool boxes = warp == kConsumerWarps;
    const int blocks_per_stage = TK >> pb_shift;
    const uint32_t box_bytes = (uint32_t)pb * 2 * D;
    const int scales_per_page = p.page_size >> sb_shift;
    int s = 0;
    uint32_t empty_parity = 1;  // a fresh barrier passes a wait on parity 1: all stages start empty
    int k = 0;
    int fills = 0;  // stages announced so far
    // where the next piece starts: stage `rel` (per head sequence, heads one after the other) of tile t of sequence sq
    long long g = g0;
    int sq = 0, t = 0;
    long long rel = 0;
    Seq cur = {0, 0, 0, 0};
    // 32 sequences' lengths at a time, one per lane
    int seq_block = -1;
    Seq ahead = {0, 0, 0, 0};
    auto fetch_seq = [&](int i) {
      if ((i >> 5) != seq_block) {
        seq_block = i >> 5;
        unsigned none = 0;
        const int mine = seq_block * 32 + lane;
        ahead = {0, 0, 0, 0};
        if (mine < S) ahead = load_seq(p, mine, RT, none);
      }
      Seq q;
      q.q_start = __shfl_sync(0xffffffffu, ahead.q_start, i & 31);
      q.q_len = __shfl_sync(0xffffffffu, ahead.q_len, i & 31);
      q.kv_len = __shfl_sync(0xffffffffu, ahead.kv_len, i & 31);
      q.tiles = __shfl_sync(0xffffffffu, ahead.tiles, i & 31);
      return q;
    };
    if (g < g1) {
      sq = share->seq[0];
      rel = g - share->base[0] * Hkv;
      cur = fetch_seq(sq);
    }
    bool alive = true;
    while (alive) {
      if (g >= g1) {
        // end-of-stream marker for the consumers
        if (!mbar_wait(bar_empty + s * 8, empty_parity, abort_flag, wait_ns)) break;
        if (lane == 0) {
          if (!boxes) metas[s] = make_int2(-1, 0);
          mbar_arrive(bar_full + s * 8);
        }
        if (!boxes) cp_async_arrive(bar_full + s * 8);
        ++fills;
        break;
      }
      // the tile that holds stage `rel`
      int lo = 0, hi = 0, n_t = 0;
      while (true) {
        if (t >= cur.tiles) {
          if (++sq >= S) break;
          cur = fetch_seq(sq);
          t = 0;
          continue;
        }
        n_t = tile_stages(p, cur, t, RT, lo, hi);
        if (rel < (long long)n_t * Hkv) break;
        rel -= (long long)n_t * Hkv;
        ++t;
      }
      if (sq >= S) {  // only if the lengths change under the call
        *abort_flag = 1;
        break;
      }
      const int h = (int)(rel / n_t), st = (int)(rel - (long long)h * n_t);
      const int take = (int)min((long long)(n_t - st), g1 - g);
      Unit u;
      u.seq = sq;
      u.row0 = t * RT;
      u.kv_begin = lo + st * TK;
      u.kv_end = st + take == n_t ? hi : lo + (st + take) * TK;
      u.q_start = cur.q_start;
      u.q_len = cur.q_len;
      u.kv_len = cur.kv_len;
      {
        const long long fs = g - st;  // the pair's first stage
        const int c0 = (int)(fs / quota), c1 = (int)((fs + n_t - 1) / quota);
        u.n_chunks = c1 - c0 + 1;
        u.chunk_idx = (int)blockIdx.x - c0;
        u.merge_idx = c0;
        // slot 2c: the piece that CTA c begins with, 2c + 1: the one that it ends with
        u.pad = fs == (long long)c0 * quota ? 2 * c0 : 2 * c0 + 1;
        u.slot = u.n_chunks == 1 ? -1 : (u.chunk_idx == 0 ? u.pad : 2 * (int)blockIdx.x);
      }
      const bool first_piece = g == g0;
      g += take;
      rel += take;
      const int ring_slot = k % kRing;
      const int32_t* tab = p.block_tables + (size_t)u.seq * p.pages_per_seq;
      // page of the block of tokens that this lane fetches; read a stage ahead, so that its latency lies under the stage before
      auto page_of = [&](int pos, int& off) {
        const int key = pos + (lane << pb_shift);
        int pi;
        if (p.page_shift >= 0) {
          pi = key >> p.page_shift;
          off = key & (p.page_size - 1);
        } else {
          pi = key / p.page_size;
          off = key - pi * p.page_size;
        }
        return lane < blocks_per_stage && key < u.kv_end ? __ldg(tab + pi) : 0;
      };
      int off_next = 0, page_next = page_of(u.kv_begin, off_next);
      bool first = true;
      for (int pos = u.kv_begin; first || pos < u.kv_end; pos += TK) {
        int nblk = (u.kv_end - pos + pb - 1) >> pb_shift;
        if (nblk > blocks_per_stage) nblk = blocks_per_stage;
        if (nblk < 0) nblk = 0;
        int page = page_next;
        const int off = off_next;
        page_next = page_of(pos + TK, off_next);
        if ((unsigned)page >= (unsigned)p.num_pages) {  // reported, and read as page 0
          if (boxes) flags |= EJK_RPA_ST_PAGE_ID;
          page = 0;
        }
        if (!mbar_wait(bar_empty + s * 8, empty_parity, abort_flag, wait_ns)) {
          alive = false;
          break;
        }
        // test hook: the stage is never announced, the consumers' wait for it must run out
        const bool withhold = (p.test_withhold & 1) && blockIdx.x == 0 && k == 0 && first;
        const uint32_t full = bar_full + s * 8;
        if (boxes && !withhold) {
          if (lane == 0) {
            if (nblk > 0) mbar_arrive_expect_tx(full, (uint32_t)nblk * box_bytes);
            else mbar_arrive(full);
          }
          __syncwarp();
          if (lane < nblk) tma_load_5d(smem_base + s * C::STAGE_BYTES + lane * box_bytes, &tmap, full, 0, off, 0, 2 * h, page);
        }
        if (!boxes && !withhold) {
          // scales of the blocks that the stage's keys lie in: K's, then V's.  Block e starts at key (e0 + e) << sb_shift, or
          // at the stage's first key; the lane that fetches that key's tokens knows its page
          const int e0 = pos >> sb_shift;
          const int last = (u.kv_end < pos + TK ? u.kv_end : pos + TK) - 1;
          const int n_e = last >= pos ? (last >> sb_shift) - e0 + 1 : 0;
          const uint32_t sdst = smem_base + C::OFF_SCALE + s * (2 * TK * 4);
          for (int e = lane; e - lane < n_e; e += 32) {
            const int from = max(((e0 + e) << sb_shift) - pos, 0);  // tokens into the stage
            const int at_lane = (from >> pb_shift) & 31;
            const int pg = __shfl_sync(0xffffffffu, page, at_lane), of = __shfl_sync(0xffffffffu, off, at_lane);
            if (e < n_e) {
              const long long at = ((long long)pg * Hkv + h) * (2 * scales_per_page) + ((of + (from & (pb - 1))) >> sb_shift);
              cp_async4(sdst + e * 4, cache.scales + at);
              cp_async4(sdst + (TK + e) * 4, cache.scales + at + scales_per_page);
            }
          }
        }
        if (!boxes && first) {
          // the piece's descriptor and query tile travel with its first stage
          if (lane == 0) {
            ItemDesc d;
            d.u = u;
            d.h = h;
            d.first = first_piece;
            ring[ring_slot] = d;
          }
          constexpr int QCH = D / 8;  // 16-byte chunks of a row: 8, 16 or 32 neighbouring lanes hold one row
          uint8_t* qdst = smem + C::OFF_Q + s * C::Q_BYTES;
          float* qfac = reinterpret_cast<float*>(smem + C::OFF_QFAC + s * RT * 4);
          const int rows_total = u.q_len * G;
#pragma unroll 4
          for (int cidx = lane; cidx < RT * QCH; cidx += 32) {
            const int r = cidx / QCH, ch = cidx % QCH;
            const int R = u.row0 + r;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (R < rows_total) {
              const int qt = R / G, g = R - qt * G;
              v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p.q) +
                                                       ((size_t)(u.q_start + qt) * p.Hq + h * G + g) * D * sizeof(T) + ch * 16));
            }
            if constexpr (!std::is_same<T, __half>::value) {
              // to f16 by a power of two that takes the row's largest element to [2^14, 2^15): exact for every element
              // above 2^-28 of it, absolute error 2^-39 of it below
              uint32_t w[4] = {v.x, v.y, v.z, v.w};
              uint32_t big = 0;
#pragma unroll
              for (int i = 0; i < 4; ++i) big = max(big, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
#pragma unroll
              for (int o = QCH / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
              int e = (int)(big >> 23);  // biased exponent of the row's largest element
              e = e == 255 ? 127 + 14 : (e < 20 ? 20 : e);  // infinities and NaN stay what they are; 2^k stays finite
              const float up = __uint_as_float((uint32_t)(254 + 14 - e) << 23);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 a = unpack2<T>(w[i]);
                w[i] = Mma<__half>::pack(a.x * up, a.y * up);
              }
              v = make_uint4(w[0], w[1], w[2], w[3]);
              if (ch == 0) qfac[r] = __uint_as_float((uint32_t)(e - 14) << 23);
            } else {
              if (ch == 0) qfac[r] = 1.f;
            }
            *reinterpret_cast<uint4*>(qdst + r * C::Q_ROW_BYTES + ch * 16) = v;
          }
        }
        __syncwarp();  // what the lanes wrote is ordered before the announcement
        ++fills;
        if (!boxes && !withhold) {
          if (lane == 0) {
            metas[s] = make_int2(ring_slot, pos);
            mbar_arrive(full);
          }
          cp_async_arrive(full);
        }
        first = false;
        if (++s == NS) {
          s = 0;
          empty_parity ^= 1u;
        }
      }
      ++k;
    }
    // Leave only after every bulk copy this warp issued has landed: wait (bounded) for the
    // consumers to drain all stages, which implies all "full" phases completed.
    for (int i = 0; i < NS; ++i) {
      if (!mbar_wait(bar_empty + s * 8, empty_parity, abort_flag, wait_ns)) break;
      if (++s == NS) {
        s = 0;
        empty_parity ^= 1u;
      }
    }
    if (*abort_flag) {
      // Giving up: the consumers no longer release stages, so wait (bounded, 2 ms per stage) for the
      // copies themselves -- the "full" phase of each of the last NS announced stages -- before this
      // CTA's shared memory can go to another CTA.
      flags |= EJK_RPA_ST_TIMEOUT;
      for (int i = 1; i <= NS && i <= fills; ++i) {
        const int f = fills - i;
        mbar_wait_quiet(bar_full + (f % NS) * 8, (uint32_t)((f / NS) & 1), 2000000ull);
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  } else {
    // =============================== consumer warps ===============================
    // Shared-memory offsets of this lane's ldmatrix rows.  Token tl of the stage sits in box tl / pb at row tl % pb; a
    // box is [K|V][DC columns][pb rows][RB bytes].  The swizzle XORs the 16-byte chunk with the row number, counted
    // in 128-byte lines: row & 7 at 128-byte rows, (row >> 1) & 3 at 64-byte rows.
    const uint32_t swz = (uint32_t)((C::RB == 128 ? (lane & 7) : ((lane & 7) >> 1))) << 4;
    const uint32_t dc_stride = (uint32_t)pb * C::RB;
    auto row_off = [&](int tl, int kv) {
      const int j = tl >> pb_shift, tp = tl & (pb - 1);
      return (uint32_t)((j * 2 + kv) * C::DC) * dc_stride + (uint32_t)tp * C::RB;
    };
    // K: two 16-token blocks, in each the matrices (tokens 0-7 | 8-15) x (16-byte chunk c | c + 1);
    // V: four transposed matrices of one chunk, tokens 8j .. 8j+7
    const uint32_t k_off0 = row_off(warp * TW + (lane & 7) + ((lane >> 3) & 1) * 8, 0);
    const uint32_t k_off1 = row_off(warp * TW + 16 + (lane & 7) + ((lane >> 3) & 1) * 8, 0);
    const uint32_t v_off = row_off(warp * TW + (lane & 7) + (lane >> 3) * 8, 1);
    const int k_dhalf = lane >> 4;

    uint32_t qf[NT][D / 32][4];  // B operands of Q.K^T: two f16 mmas per 32-byte chunk of K
    float acc[NT][KT][4];
    float m_run[NT][2], l_run[NT][2], q_fac[NT][2];
    int pos_r[NT][2], lo_r[NT][2];
    int pos_min = 0, lo_max = 0, lo_min = -1;
    bool one_token = true;  // the tile's rows are one query token's: they see the same keys
    float v_norm = 1.f;  // power of two that the V scales are multiplied by
    bool mixed = false;  // some row has not seen a key that another has
    bool far = false;    // ... and scales lie far apart: the piece's rows are computed one by one at its end
    int s = 0;
    uint32_t full_parity = 0, c_parity = 0;
    int pieces = 0;
    int arrived = 0, owed = 0;  // bit 0 / 1 = the CTA's first / another shared piece has been counted; its group not yet

    auto consumer_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_c);
      const bool ok = mbar_wait(bar_c, c_parity, abort_flag, wait_ns);
      c_parity ^= 1u;
      return ok;
    };

    // some row of the tile does not see all of the warp's keys
    auto masked = [&](int key0, int kv_end) { return key0 + TW > kv_end || (key0 + TW - 1 > pos_min) || (key0 <= lo_max); };
    // is some V scale of the warp's keys far below the largest that any row has seen?
    auto far_scales = [&](int pos, int kv_end) {
      const int key = pos + warp * TW + lane;
      const float* vs = reinterpret_cast<const float*>(smem + C::OFF_SCALE + s * (2 * TK * 4)) + TK;
      const bool seen = key < kv_end && key > lo_min;
      const float v = seen ? vs[(key >> sb_shift) - (pos >> sb_shift)] : 0.f;
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
      const float unit = top * v_norm >= (float)(2 << kVBits) ? scale_unit(top) : v_norm;
      return __any_sync(0xffffffffu, seen && v * unit < kFar) != 0;
    };
    // The warp's 32 keys of a stage
    auto stage = [&](int pos, int kv_end) {
      const int key0 = pos + warp * TW;
      const uint32_t sbase = smem_base + s * C::STAGE_BYTES;
      // ---- S^T[32 tokens x rows] = K . Q^T as two 16-token blocks
      float sc[NT][2][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][b][e] = 0.f;
#pragma unroll
      for (int kt = 0; kt < D / 32; ++kt) {
        const int c16 = kt * 2;  // 16-byte chunk of the token's row; + k_dhalf at run time
        const uint32_t coff = (uint32_t)(c16 / CH) * dc_stride + ((((uint32_t)(c16 % CH) | (uint32_t)k_dhalf) << 4) ^ swz);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          // a[0] = (token g, bytes 4t..4t+3 of the chunk), a[1] = token g+8, a[2] / a[3] = the next chunk.  The low two
          // bytes of a register become k slots 2t, 2t+1, the high two k slots 8+2t, 8+2t+1 of one f16 mma -- the
          // query fragments were loaded in the same order
          uint32_t a[4];
          ldmatrix_x4(a, sbase + (b ? k_off1 : k_off0) + coff);
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) Code::widen(a[i], lo[i], hi[i]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(sc[nt][b], lo[0], lo[1], hi[0], hi[1], qf[nt][kt][0], qf[nt][kt][1]);
            mma_f16(sc[nt][b], lo[2], lo[3], hi[2], hi[3], qf[nt][kt][2], qf[nt][kt][3]);
          }
        }
      }
      // ---- scales of this lane's four tokens
      const float* ks_s = reinterpret_cast<const float*>(smem + C::OFF_SCALE + s * (2 * TK * 4));
      const float* vs_s = ks_s + TK;
      const int e0 = pos >> sb_shift;
      float ks[4], vs[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + (lane >> 2) + i * 8;
        const int e = (key >> sb_shift) - e0;
        ks[i] = ks_s[e];
        // no row sees a key from kv_end on, or one that the window of the tile's first row has left behind
        vs[i] = (key < kv_end && key > lo_min) ? vs_s[e] : 0.f;
      }
      const bool tail = key0 + TW > kv_end;  // tokens past the chunk end: stale or unowned bytes
      const bool edge = tail || key0 <= lo_min;
      const bool need_mask = masked(key0, kv_end);
      // the power of two by the largest V scale of the warp's 32 keys (positive floats order as integers)
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])))));
      if (top * v_norm >= (float)(2 << kVBits)) {
        // a larger scale than any before: the accumulators go along
        const float v_new = scale_unit(top);
        const float f = v_new * power_of_two_inverse(v_norm);  // 0 where the old terms are below anything that counts
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < KT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][mt][i] *= f;
        v_norm = v_new;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) vs[i] *= v_norm;
      bool grow = false;
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = e & 1;
            float x = sc[nt][b][e] * (q_fac[nt][j] * ks[b * 2 + (e >> 1)]);
            if (p.cap != 0.f) x = p.cap_log2 * soft_cap_tanh(x);
            if (need_mask) {
              // a 128-token stage can straddle the end of a chunk (chunks are cut at multiples of 64): keys from
              // kv_end on belong to the next chunk, or to nobody
              const int key = key0 + b * 16 + (lane >> 2) + (e >> 1) * 8;
              if (key > pos_r[nt][j] || key <= lo_r[nt][j] || key >= kv_end) x = -INFINITY;
            }
            sc[nt][b][e] = x;
          }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v = fmaxf(fmaxf(sc[nt][0][j], sc[nt][0][j + 2]), fmaxf(sc[nt][1][j], sc[nt][1][j + 2]));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          mx[nt][j] = v;
          // lazy rescaling: keep the old reference maximum unless the new one is 2^8 larger
          grow |= (v > m_run[nt][j] + kLazyRescale) || (m_run[nt][j] == -INFINITY && v > -INFINITY);
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float alpha[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const bool g = (mx[nt][j] > m_run[nt][j] + kLazyRescale) || (m_run[nt][j] == -INFINITY && mx[nt][j] > -INFINITY);
            const float m_new = g ? mx[nt][j] : m_run[nt][j];
            alpha[j] = g ? fast_exp2(m_run[nt][j] - m_new) : 1.f;  // exp2(-inf) = 0 on the first tile
            m_run[nt][j] = m_new;
            l_run[nt][j] *= alpha[j];
          }
#pragma unroll
          for (int mt = 0; mt < KT; ++mt) {
            acc[nt][mt][0] *= alpha[0];
            acc[nt][mt][1] *= alpha[1];
            acc[nt][mt][2] *= alpha[0];
            acc[nt][mt][3] *= alpha[1];
          }
        }
      }
      // ---- probabilities; times the V scale to f16, transposed into the B fragments of P.V
      uint32_t pbf[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float m_use = (m_run[nt][j] == -INFINITY) ? 0.f : m_run[nt][j];
            const float p0 = fast_exp2(sc[nt][b][j] - m_use);
            const float p1 = fast_exp2(sc[nt][b][j + 2] - m_use);
            l_run[nt][j] += p0 + p1;
            sc[nt][b][j] = p0 * vs[b * 2];
            sc[nt][b][j + 2] = p1 * vs[b * 2 + 1];
          }
          pbf[nt][b * 2] = movmatrix_trans(Mma<__half>::pack(sc[nt][b][0], sc[nt][b][1]));
          pbf[nt][b * 2 + 1] = movmatrix_trans(Mma<__half>::pack(sc[nt][b][2], sc[nt][b][3]));
        }
      }
      // ---- V^T fragments: four transposed 8-token matrices of one 16-byte chunk; register j holds, for the two
      // head-dim lanes 2g and 2g+1, tokens 8j + 2t (low half) and 8j + 2t + 1 (high half): rows g and g+8 of the mma
      // stand for lanes 16mt + 2g and + 1.  The bytes of keys that no row sees are cleared, so that 0 * (stale
      // NaN) cannot reach the accumulators.
      uint32_t vmask[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
      if (edge) {
        const int t0 = key0 + (lane & 3) * 2;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int a = t0 + 8 * j;
          vmask[j] = (a < kv_end && a > lo_min ? 0x0000ffffu : 0u) | (a + 1 < kv_end && a + 1 > lo_min ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int mt = 0; mt < KT; ++mt) {
        uint32_t r[4];
        ldmatrix_x4_trans(r, sbase + v_off + (uint32_t)(mt / CH) * dc_stride + (((uint32_t)(mt % CH) << 4) ^ swz));
        if (edge) {
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] &= vmask[j];
        }
        uint32_t even[4], odd[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) Code::widen_interleaved(r[j], even[j], odd[j]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(acc[nt][mt], even[0], odd[0], even[1], odd[1], pbf[nt][0], pbf[nt][1]);
          mma_f16(acc[nt][mt], even[2], odd[2], even[3], odd[3], pbf[nt][2], pbf[nt][3]);
        }
      }
    };

    while (true) {
      // the stages of a piece
      int2 meta;
      bool end = false;
      while (true) {
        if (!mbar_wait(bar_full + s * 8, full_parity, abort_flag, wait_ns)) {
          end = true;
          break;
        }
        meta = metas[s];
        end = meta.x < 0;
        if (end) break;
        const Unit u = ring[meta.x].u;
        const int pos = meta.y;
        const int rows_total = u.q_len * G;
        int n_rows = rows_total - u.row0;
        if (n_rows > RT) n_rows = RT;

        if (pos == u.kv_begin) {
          const uint8_t* qs = smem + C::OFF_Q + s * C::Q_BYTES;
          const float* qfac = reinterpret_cast<const float*>(smem + C::OFF_QFAC + s * RT * 4);
          const float to_log2 = p.cap != 0.f ? p.inv_cap_scale : p.scale_log2;
          const int base = u.kv_len - u.q_len;
          pos_min = base + u.row0 / G;
          one_token = (u.row0 + n_rows - 1) / G == u.row0 / G;
          v_norm = __uint_as_float((127u + 125u) << 23);  // no scale met yet: the largest power of two (see below)
          mixed = far = false;
          lo_max = (p.window > 0) ? (base + (u.row0 + n_rows - 1) / G - p.window) : -1;
          lo_min = (p.window > 0) ? pos_min - p.window : -1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            // elements 32kt + 4t .. +3 (first mma of the chunk) and 32kt + 16 + 4t .. +3 (second)
            const uint8_t* qrow = qs + (nt * 8 + (lane >> 2)) * C::Q_ROW_BYTES + (lane & 3) * 8;
#pragma unroll
            for (int kt = 0; kt < D / 32; ++kt) {
              const uint2 a = *reinterpret_cast<const uint2*>(qrow + kt * 64);
              const uint2 b = *reinterpret_cast<const uint2*>(qrow + kt * 64 + 32);
              qf[nt][kt][0] = a.x;
              qf[nt][kt][1] = a.y;
              qf[nt][kt][2] = b.x;
              qf[nt][kt][3] = b.y;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = nt * 8 + (lane & 3) * 2 + j;
              const int R = u.row0 + r;
              const int ps = (R < rows_total) ? base + R / G : -1;
              pos_r[nt][j] = ps;
              lo_r[nt][j] = (p.window > 0) ? ps - p.window : -1;
              q_fac[nt][j] = qfac[r] * to_log2;
              m_run[nt][j] = -INFINITY;
              l_run[nt][j] = 0.f;
            }
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nt][kt][e] = 0.f;
          }
        }

        const int key0 = pos + warp * TW;
        if (key0 < u.kv_end) {
          if (!one_token) {
            mixed |= masked(key0, u.kv_end);
            if (mixed) far |= far_scales(pos, u.kv_end);
          }
          stage(pos, u.kv_end);
        }
        if (pos + TK >= u.kv_end) break;
        // this warp is done with the stage's bytes (query fragments are in registers by now)
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + s * 8);
        if (++s == NS) {
          s = 0;
          full_parity ^= 1u;
        }
      }
      if (end) break;
      const ItemDesc& it = ring[meta.x];
      const Unit u = it.u;
      const int h = it.h;
      const bool first_piece = it.first != 0;
      const int pos = meta.y;
      int n_rows = u.q_len * G - u.row0;
      if (n_rows > RT) n_rows = RT;
      if (pos + TK >= u.kv_end) {
        // ---- end of the piece.  The warps' accumulators meet in the memory of its last stage: with the first barrier every
        // warp is done with the stage and has published its rows' (m, l), with the second all accumulators are there; from
        // then on the warps go their own ways, each with its own rows.
        float2* ml = mlbuf + (pieces & 1) * (kConsumerWarps * RT);  // two, for a warp that is a piece ahead
        ++pieces;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float l = l_run[nt][j];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            // (the sum's sign: the rows have to be computed one by one)
            if (lane < 4) ml[warp * RT + nt * 8 + lane * 2 + j] = make_float2(m_run[nt][j], far ? -l : l);
          }
        if (!consumer_sync()) break;
        // accumulators relative to the rows' common maximum, without the power of two that this warp took the row's V scales
        // by.  Row r, head-dim lane d of warp w is at [w][r][d], with d's 16-lane block XORed by r / 2 against bank conflicts
        float* sum = reinterpret_cast<float*>(smem + s * C::STAGE_BYTES);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = nt * 8 + (lane & 3) * 2 + j;
            float mt = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumerWarps; ++w) mt = fmaxf(mt, ml[w * RT + r].x);
            const float f = fast_exp2(m_run[nt][j] - ((mt == -INFINITY) ? 0.f : mt)) * power_of_two_inverse(v_norm);
            // accumulator rows g / g+8 of block mt are head-dim lanes 16mt + 2g / + 1 (see the V fragments)
            float* row = sum + (warp * RT + r) * D + (lane >> 2) * 2;
#pragma unroll
            for (int mt16 = 0; mt16 < KT; ++mt16)
              *reinterpret_cast<float2*>(row + (mt16 ^ (lane & 3)) * 16) = make_float2(acc[nt][mt16][j] * f, acc[nt][mt16][j + 2] * f);
          }
        if (!consumer_sync()) break;
        constexpr int VPL = D / 32;   // columns per lane
        constexpr int RPW = RT / kConsumerWarps;  // rows per warp: warp, warp + 4, ...
        T* out = reinterpret_cast<T*>(p.out);
        auto store_row = [&](int r, float m_tot, float l_tot, const float (&o)[VPL]) {
          const int R = u.row0 + r;
          const int qt = R / G, gq = R - qt * G;
          const int hq = h * G + gq;
          float scl = 1.f, l_fin = l_tot;
          if (p.num_sinks > 0) {
            // attention sinks join the denominator only
            const int srow = (p.sink_rows == p.Hq) ? hq : (p.sink_rows == Hkv ? h : 0);
            const float* sk = p.sinks + (size_t)srow * p.num_sinks;
            float sm = -INFINITY;
            for (int i = 0; i < p.num_sinks; ++i) sm = fmaxf(sm, sk[i] * kLog2e);
            const float m_fin = fmaxf(m_tot, sm);
            const float mf = (m_fin == -INFINITY) ? 0.f : m_fin;
            scl = fast_exp2(m_tot - mf);
            l_fin = l_tot * scl;
            for (int i = 0; i < p.num_sinks; ++i) l_fin += fast_exp2(sk[i] * kLog2e - mf);
          }
          scl = (l_fin > 0.f) ? scl / l_fin : 0.f;
          uint32_t* dst = reinterpret_cast<uint32_t*>(out + ((size_t)(u.q_start + qt) * p.Hq + hq) * D + lane * VPL);
#pragma unroll
          for (int i = 0; i < VPL; i += 2) dst[i / 2] = Mma<T>::pack(o[i] * scl, o[i + 1] * scl);
        };
        auto store_part = [&](int slot, int r, float m_tot, float l_tot, const float (&o)[VPL]) {
          float* dst = p.part_o + ((size_t)slot * RT + r) * D + lane * VPL;
#pragma unroll
          for (int i = 0; i < VPL; i += 2) *reinterpret_cast<float2*>(dst + i) = make_float2(o[i], o[i + 1]);
          if (lane == 0) p.part_ml[(size_t)slot * RT + r] = make_float2(m_tot, l_tot);
        };
#pragma unroll
        for (int ri = 0; ri < RPW; ++ri) {
          const int r = warp + ri * kConsumerWarps;
          float m_tot = -INFINITY, l_tot = 0.f;
          uint32_t any_far = 0;
#pragma unroll
          for (int w = 0; w < kConsumerWarps; ++w) m_tot = fmaxf(m_tot, ml[w * RT + r].x);
          const float mu = (m_tot == -INFINITY) ? 0.f : m_tot;
#pragma unroll
          for (int w = 0; w < kConsumerWarps; ++w) {
            const float l = ml[w * RT + r].y;
            any_far |= __float_as_uint(l) >> 31;
            l_tot += fabsf(l) * fast_exp2(ml[w * RT + r].x - mu);
          }
          const int col = lane * VPL;
          const float* src = sum + r * D + (((col >> 4) ^ ((r >> 1) & 3)) << 4) + (col & 15);
          float o[VPL];
#pragma unroll
          for (int i = 0; i < VPL; ++i) o[i] = 0.f;
#pragma unroll
          for (int w = 0; w < kConsumerWarps; ++w)
#pragma unroll
            for (int i = 0; i < VPL; i += 2) {
              const float2 v = *reinterpret_cast<const float2*>(src + w * RT * D + i);
              o[i] += v.x;
              o[i + 1] += v.y;
            }
          if (r >= n_rows) continue;
          if (__builtin_expect(any_far != 0, 0)) {
            const int R = u.row0 + r, qt = R / G;
            const int at = u.kv_len - u.q_len + qt;  // the row's position
            FarRow f;
            f.q = reinterpret_cast<const T*>(p.q) + ((size_t)(u.q_start + qt) * p.Hq + h * G + (R - qt * G)) * D;
            f.table = p.block_tables + (size_t)u.seq * p.pages_per_seq;
            f.pages = cache.pages;
            f.scales = cache.scales;
            f.num_pages = p.num_pages;
            f.page_size = p.page_size;
            f.Hkv = Hkv;
            f.h = h;
            f.block_shift = cache.block_shift;
            f.key0 = max(u.kv_begin, p.window > 0 ? at - p.window + 1 : 0);
            f.key1 = min(u.kv_end, at + 1);
            f.scale_log2 = p.scale_log2;
            f.cap_log2 = p.cap_log2;
            f.inv_cap_scale = p.inv_cap_scale;
            far_row<T, Code, D>(&f);
            m_tot = f.m;
            l_tot = f.l;
#pragma unroll
            for (int i = 0; i < VPL; ++i) o[i] = f.o[i];
          }
          if (u.slot < 0) store_row(r, m_tot, l_tot, o);
          else store_part(u.slot, r, m_tot, l_tot, o);
        }
        // the stage can go back (its memory was written by ordinary stores, the next box comes through the async proxy)
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + s * 8);
        if (u.slot >= 0) {
          // Last-arriver merge of this warp's rows: publish the part, take a ticket; whoever draws the last one combines the
          // parts, in part order, so that the result does not depend on who that is.  Nobody ever waits for another CTA.
          const int c0 = u.merge_idx, bit = first_piece ? 1 : 2;
          int* tickets = p.tickets + warp * 3 * n_cta;
          bool groups = false;
          while (true) {
            __threadfence();
            __syncwarp();
            Arrival a = {0, 0, 0, true};
            if (lane == 0) a = groups ? arrive_group(tickets, n_cta, c0, u.n_chunks) : arrive_part(tickets, n_cta, c0, u.chunk_idx, u.n_chunks);
            const int count = __shfl_sync(0xffffffffu, a.count, 0), stride = __shfl_sync(0xffffffffu, a.stride, 0);
            const int part0 = __shfl_sync(0xffffffffu, a.part0, 0);
            const bool last = __shfl_sync(0xffffffffu, (int)a.last, 0) != 0;
            arrived |= bit;
            owed = count && !last ? owed | bit : owed & ~bit;
            if (count == 0) break;
            __threadfence();
            auto slot_of = [&](int i) {
              const int part = part0 + i * stride;
              return part == 0 ? u.pad : 2 * (c0 + part);
            };
#pragma unroll 1
            for (int r = warp; r < n_rows; r += kConsumerWarps) {
              // lane i holds part i's maximum and sum (count <= 32)
              const float2 mlp = lane < count ? __ldcg(&p.part_ml[(size_t)slot_of(lane) * RT + r]) : make_float2(-INFINITY, 0.f);
              float m_tot = mlp.x;
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) m_tot = fmaxf(m_tot, __shfl_xor_sync(0xffffffffu, m_tot, o));
              const float mu = (m_tot == -INFINITY) ? 0.f : m_tot;
              const float f_mine = fast_exp2(mlp.x - mu);
              float l_tot = mlp.y * f_mine;
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) l_tot += __shfl_xor_sync(0xffffffffu, l_tot, o);
              float o[VPL];
#pragma unroll
              for (int i = 0; i < VPL; ++i) o[i] = 0.f;
              for (int i0 = 0; i0 < count; i0 += kMergeInFlight) {
                float2 v[kMergeInFlight][VPL / 2];
#pragma unroll
                for (int j = 0; j < kMergeInFlight; ++j) {
                  const float* src = p.part_o + ((size_t)slot_of(min(i0 + j, count - 1)) * RT + r) * D + lane * VPL;
#pragma unroll
                  for (int i = 0; i < VPL / 2; ++i) v[j][i] = __ldcg(reinterpret_cast<const float2*>(src) + i);
                }
#pragma unroll
                for (int j = 0; j < kMergeInFlight; ++j) {
                  const float f = __shfl_sync(0xffffffffu, f_mine, min(i0 + j, 31));
                  if (i0 + j < count) {
#pragma unroll
                    for (int i = 0; i < VPL / 2; ++i) {
                      o[2 * i] += v[j][i].x * f;
                      o[2 * i + 1] += v[j][i].y * f;
                    }
                  }
                }
              }
              if (last) store_row(r, m_tot, l_tot, o);
              else store_part(slot_of(0), r, m_tot, l_tot, o);  // a group: its sum takes the place of its first part
            }
            if (last) break;
            groups = true;
          }
        }
      } else {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + s * 8);
      }
      if (++s == NS) {
        s = 0;
        full_parity ^= 1u;
      }
    }
    if (*abort_flag) flags |= EJK_RPA_ST_TIMEOUT;
    if (*abort_flag && lane == 0 && g0 < g1) {
      // Giving up: the shared pieces that were not counted are counted now, with no data, so that the counters are zero again
      // after the call (the outputs are invalid, which the status says).
      for (int e = 0; e < 2; ++e) {
        const long long g = e ? g1 - 1 : g0;
        unsigned none = 0;
        const Seq q = load_seq(p, share->seq[e], RT, none);
        long long rel = g - share->base[e] * Hkv;
        int lo, hi, n_t = 1;
        for (int t = 0; t < q.tiles; ++t) {
          n_t = tile_stages(p, q, t, RT, lo, hi);
          if (rel < (long long)n_t * Hkv) break;
          rel -= (long long)n_t * Hkv;
        }
        const long long fs = g - rel % n_t;
        const int c0 = (int)(fs / quota), c1 = (int)((fs + n_t - 1) / quota);
        const int bit = fs <= g0 ? 1 : 2;  // the CTA's first piece, or another
        if (c0 == c1) continue;
        bool group_next = (owed & bit) != 0;
        if (!(arrived & bit)) {
          const Arrival a = arrive_part(p.tickets + warp * 3 * n_cta, n_cta, c0, (int)blockIdx.x - c0, c1 - c0 + 1);
          group_next = a.count && !a.last;
        }
        if (group_next) arrive_group(p.tickets + warp * 3 * n_cta, n_cta, c0, c1 - c0 + 1);
        arrived |= bit;
        owed &= ~bit;
      }
    }
  }
  if (flags && p.status) atomicOr(reinterpret_cast<unsigned*>(p.status), flags);
  {
    // rows of no sequence: in front of the first, behind the last, and those of sequences whose offsets are refused.  Between
    // the first offset and the last every row lies between two neighbouring offsets, whatever their order: none is left out
    const size_t row_bytes = (size_t)p.Hq * D * sizeof(T);
    const int head = __ldg(p.query_start_loc), tail = __ldg(p.query_start_loc + S);
    zero_tail_rows(p.out, 0, min(max(head, 0), p.T), row_bytes);
    zero_tail_rows(p.out, min(max(tail, 0), p.T), p.T, row_bytes);
    if (*bad_offsets) {
      for (int i = 0; i < S; ++i) {
        const int q0 = __ldg(p.query_start_loc + i), q1 = __ldg(p.query_start_loc + i + 1);
        if (bad_rows(q0, q1, p.T)) zero_tail_rows(p.out, max(q0, 0), min(q1, p.T), row_bytes);
      }
    }
  }
  // In a mixed batch this grid is a programmatic dependent of the prefill-tile grid and never waited for it
  // (the two write different rows).  Whatever follows in the stream, though, is only ordered after THIS grid:
  // one thread per CTA now waits for the prefill grid, so this grid cannot complete before it, and a later
  // kernel (a reader of `out`, the next call's planner) is ordered after both.  All prefill CTAs are resident
  // before this grid starts (it is released when each of them has seen the plan), so the wait cannot starve them.
  if ((p.pdl & 1) && tid == 0) pdl_wait();
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    fn = reinterpret_cast<EncodeFn>(ptr);
  }
  return fn;
}

template <typename T, typename Code, int D, int NT, int NS>
cudaError_t launch_one(const Params& p, const Q8Cache& c, const CUtensorMap& map, int n_sm, cudaStream_t stream, bool pdl) {
  using C = Cfg<D, NT, NS>;
  auto kern = q8_splitkv_kernel<T, Code, D, NT, NS>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  return launch_kernel(kern, dim3(n_sm * C::CTAS), dim3(kThreads), C::SMEM_BYTES, stream, pdl, map, p, c);
}

template <typename T, typename Code>
cudaError_t dispatch(const Params& p, const Q8Cache& c, const CUtensorMap& map, int n_sm, cudaStream_t stream, bool pdl) {
  const bool wide = p.rows_per_tile == 16;
  switch (p.D) {
    case 64:
      return wide ? launch_one<T, Code, 64, 2, 5>(p, c, map, n_sm, stream, pdl) : launch_one<T, Code, 64, 1, 5>(p, c, map, n_sm, stream, pdl);
    case 128:
      return wide ? launch_one<T, Code, 128, 2, 5>(p, c, map, n_sm, stream, pdl) : launch_one<T, Code, 128, 1, 3>(p, c, map, n_sm, stream, pdl);
    case 256:
      return wide ? launch_one<T, Code, 256, 2, 2>(p, c, map, n_sm, stream, pdl) : launch_one<T, Code, 256, 1, 3>(p, c, map, n_sm, stream, pdl);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

bool q8_tma_supported(int page_size) {
  // boxes are whole 8-token groups of one page: the period of the swizzle
  return page_size >= 8 && page_size % 8 == 0 && encode_fn() != nullptr;
}

// kv_pages as a tensor map, innermost first: one swizzle span of bytes | token in page | column of head_dim | head and K or
// V | page.  One box is `box_tokens` tokens of one head, K and V.
cudaError_t q8_tensor_map(CUtensorMap* map, const Q8Cache& c, int box_tokens) {
  EncodeFn enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t D = c.D, rb = c.D < 128 ? c.D : 128, page = c.page_size, planes = 2ull * c.Hkv;
  cuuint64_t dims[5] = {rb, page, D / rb, planes, (cuuint64_t)c.num_pages};
  cuuint64_t strides[4] = {D, rb, page * D, planes * page * D};
  cuuint32_t box[5] = {(cuuint32_t)rb, (cuuint32_t)box_tokens, (cuuint32_t)(D / rb), 2, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, c.pages, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         rb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t launch_q8_splitkv(const Params& p, const Q8Cache& c, int dtype, int code, int n_sm, cudaStream_t stream, bool pdl) {
  CUtensorMap map;
  if (cudaError_t e = q8_tensor_map(&map, c, p.tma_block_tokens); e != cudaSuccess) return e;
  if (code == EJK_Q8_I8)
    return dtype == EJK_RPA_BF16 ? dispatch<__nv_bfloat16, CodeI8>(p, c, map, n_sm, stream, pdl)
                                 : dispatch<__half, CodeI8>(p, c, map, n_sm, stream, pdl);
  return dtype == EJK_RPA_BF16 ? dispatch<__nv_bfloat16, CodeE4M3>(p, c, map, n_sm, stream, pdl)
                               : dispatch<__half, CodeE4M3>(p, c, map, n_sm, stream, pdl);
}

}  // namespace ejk
