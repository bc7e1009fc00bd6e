// Work list of the tensor-tile kernel (q8_prefill.cu), from the lengths on the device: one item per 256 or 128 query rows of a
// sequence with many of them, longest first, with the running sum of their 64-token KV stages.
//
// It runs before the kernel that it feeds, so its latency is on the path: one block, one pass over the sequences and one over the
// items, a bitonic sort of the items in shared memory (their order decides where the KV split cuts and therefore the last bit of a
// result, so it may not depend on thread timing).  More items than fit the sort keep the order of the sequences, each
// sequence's items from its end, where they are longest: with thousands of items the order no longer decides when the last one ends.
// 24 sequences 9 us, 4 sequences with 96 items 10 us (the planner of the 16-bit operator, which also lists the decode rows and
// orders the tiles with one warp: 12 and 28 us).
#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr int kThreads = 1024;
constexpr int kSortItems = 2048;
constexpr int kSeqs = 1024;  // sequences per round

struct SeqTiles {
  int q_start, q_len, kv_len, rows;
  bool tiles;
};
__device__ __forceinline__ SeqTiles load_seq(const Params& p, int s, unsigned& flags) {
  const int q0 = p.query_start_loc[s], q1 = p.query_start_loc[s + 1];
  int kv = p.context_lens[s];
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
  return {q0, ql, kv, ql * p.G, ql * p.G >= p.prefill_min_rows};
}
// keys that some row of [r0, r0 + n) of a sequence sees; lo is rounded down to a stage
__device__ __forceinline__ void key_range(const Params& p, const SeqTiles& q, int r0, int n, int& lo, int& hi) {
  const int r_last = min(r0 + n, q.rows) - 1;
  const int base = q.kv_len - q.q_len;
  hi = max(base + r_last / p.G + 1, 0);
  lo = p.window > 0 ? max(base + r0 / p.G - p.window + 1, 0) / kTileTokens * kTileTokens : 0;
  hi = max(hi, lo);
}

// exclusive sum over the block and the total
__device__ int block_scan(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s_warp of an earlier scan has been read
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int y = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    s_warp[lane] = y;
  }
  __syncthreads();
  total = s_warp[31];
  return x - v + (warp ? s_warp[warp - 1] : 0);
}

__global__ void __launch_bounds__(kThreads) q8_plan_kernel(const Params p, int n_cta) {
  pdl_trigger();
  pdl_wait();
  __shared__ int s_warp[32];
  __shared__ int s_first[kSeqs];
  __shared__ unsigned long long s_key[kSortItems];
  __shared__ unsigned long long s_decode_keys;
  __shared__ int s_items[2];
  const int tid = threadIdx.x;
  unsigned flags = 0;
  int S = p.num_seqs[0];
  if (S > p.S_max) {
    flags |= EJK_RPA_ST_NUM_SEQS;
    S = p.S_max;
  }
  if (S < 0) S = 0;
  if (tid == 0) s_decode_keys = 0;
  if (tid < 2) s_items[tid] = 0;
  __syncthreads();

  // ---- how many items there would be of 256 and of 128 rows, and the keys that the split-KV kernel will stream
  {
    int n256 = 0, n128 = 0;
    unsigned long long keys = 0;
    for (int s = tid; s < S; s += kThreads) {
      unsigned none = 0;
      const SeqTiles q = load_seq(p, s, none);
      if (q.tiles) {
        n256 += (q.rows + 255) >> 8;
        n128 += (q.rows + 127) >> 7;
      } else if (q.rows > 0) {
        int lo, hi;
        key_range(p, q, 0, q.rows, lo, hi);
        keys += (unsigned long long)(hi - lo) * (unsigned)((q.rows + p.rows_per_tile - 1) / p.rows_per_tile);
      }
    }
    if (n256) atomicAdd(&s_items[0], n256);
    if (n128) atomicAdd(&s_items[1], n128);
    if (keys) atomicAdd(&s_decode_keys, keys);
  }
  __syncthreads();
  // Rows of an item: an item of 128 takes about 0.6 of the time of one of 256 (one tile's softmax warps have the SM to
  // themselves), which pays where it does not cost rounds over the SMs
  const long long rounds256 = ((long long)s_items[0] * p.Hkv + n_cta - 1) / n_cta, rounds128 = ((long long)s_items[1] * p.Hkv + n_cta - 1) / n_cta;
  const bool half = rounds128 * 5 < rounds256 * 8;
  const int item_rows = half ? kPrefillRows : 2 * kPrefillRows;
  const int n_items = half ? s_items[1] : s_items[0];
  const bool fits = n_items <= p.max_punits;
  if (!fits) {
    // only where sequences overlap: nothing is listed, and the rows that the list would have served are zero
    flags |= EJK_RPA_ST_INTERNAL;
    for (int s = 0; s < S; ++s) {
      const SeqTiles q = load_seq(p, s, flags);
      if (!q.tiles) continue;
      uint4* dst = reinterpret_cast<uint4*>(p.out) + (size_t)q.q_start * p.Hq * (p.D / 8);
      const size_t n16 = (size_t)q.q_len * p.Hq * (p.D / 8);
      for (size_t i = tid; i < n16; i += kThreads) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const bool sorted = n_items <= kSortItems;
  int n_sort = 1;
  while (n_sort < n_items) n_sort <<= 1;
  for (int i = tid; sorted && i < n_sort; i += kThreads) s_key[i] = ~0ull;

  auto item_of = [&](const SeqTiles& q, int s, int t) {
    Unit u;
    u.seq = s;
    u.row0 = t * item_rows;
    key_range(p, q, u.row0, item_rows, u.kv_begin, u.kv_end);
    u.slot = item_rows;  // the kernel's second tile has rows only in items of two
    u.q_start = q.q_start;
    u.q_len = q.q_len;
    u.kv_len = q.kv_len;
    u.merge_idx = -1;
    u.chunk_idx = 0;
    u.n_chunks = 1;
    u.pad = 0;
    return u;
  };
  auto store = [&](int at, const Unit& u) {
    int4* d = reinterpret_cast<int4*>(p.punits + at);
    d[0] = make_int4(u.seq, u.row0, u.kv_begin, u.kv_end);
    d[1] = make_int4(u.slot, u.q_start, u.q_len, u.kv_len);
    d[2] = make_int4(u.merge_idx, u.chunk_idx, u.n_chunks, u.pad);
  };

  // ---- the items, one thread each: a binary search over the round's sums finds the sequence
  int base = 0;
  for (int s0 = 0; s0 < S && fits; s0 += kSeqs) {
    const int s = s0 + tid;
    int mine = 0;
    if (s < S) {
      const SeqTiles q = load_seq(p, s, flags);
      if (q.q_len > q.kv_len) flags |= EJK_RPA_ST_QLEN;
      mine = q.tiles ? (q.rows + item_rows - 1) / item_rows : 0;
    }
    int total;
    const int first = block_scan(mine, s_warp, total);
    s_first[tid] = first;
    __syncthreads();
    const int n_here = min(S - s0, kSeqs);
    for (int j = tid; j < total; j += kThreads) {
      int a = 0, b = n_here;
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (s_first[mid] <= j) a = mid;
        else b = mid;
      }
      unsigned none = 0;
      const SeqTiles q = load_seq(p, s0 + a, none);
      const int n = (q.rows + item_rows - 1) / item_rows;
      const int t = n - 1 - (j - s_first[a]);  // from the sequence's end
      const Unit u = item_of(q, s0 + a, t);
      if (sorted) {
        // longest first, ties in the order of the sequences
        const unsigned stages = (unsigned)(u.kv_end - u.kv_begin + kTileTokens - 1) / kTileTokens;
        s_key[base + j] = ((unsigned long long)(0xffffffu - min(stages, 0xffffffu)) << 40) | (unsigned long long)(base + j);
      }
      store(base + j, u);
    }
    base += total;
    __syncthreads();
  }
  if (sorted && fits && n_items > 1) {
    for (int k = 2; k <= n_sort; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int i = tid; i < n_sort; i += kThreads) {
          const int o = i ^ j;
          if (o > i) {
            const unsigned long long x = s_key[i], y = s_key[o];
            if ((x > y) == ((i & k) == 0)) {
              s_key[i] = y;
              s_key[o] = x;
            }
          }
        }
      }
    }
    __syncthreads();
    // into that order: every thread takes its items off the list before any is overwritten
    Unit u[kSortItems / kThreads];
#pragma unroll
    for (int r = 0; r < kSortItems / kThreads; ++r) {
      const int i = tid + r * kThreads;
      if (i < n_items) {
        const int4* src = reinterpret_cast<const int4*>(p.punits + (int)(s_key[i] & 0xffffffu));
        *reinterpret_cast<int4*>(&u[r].seq) = src[0];
        *reinterpret_cast<int4*>(&u[r].slot) = src[1];
        *reinterpret_cast<int4*>(&u[r].merge_idx) = src[2];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems / kThreads; ++r) {
      const int i = tid + r * kThreads;
      if (i < n_items) store(i, u[r]);
    }
    __syncthreads();
  }

  // ---- running sum of the stages, in the order of the list; the parts' counters
  int running = 0;
  for (int i0 = 0; i0 < n_items && fits; i0 += kThreads) {
    const int i = i0 + tid;
    int v = 0;
    if (i < n_items) {
      const int len = p.punits[i].kv_end - p.punits[i].kv_begin;
      v = len > 0 ? (len + kTileTokens - 1) / kTileTokens : 1;
    }
    int total;
    const int before = block_scan(v, s_warp, total);
    if (p.prefill_split && i < n_items) p.pprefix[i] = running + before;
    running += total;
  }
  if (p.prefill_split) {
    if (tid == 0) p.pprefix[fits ? n_items : 0] = running;
    const int n_pt = (fits ? n_items : 0) * p.Hkv * (p.prefill_item_rows / kPrefillRows) * 4;
    for (int i = tid; i < n_pt; i += kThreads) p.ptickets[i] = 0;
  }
  if (tid == 0) {
    p.header[kHdrPrefillQueue] = 0;
    p.header[kHdrNumPrefill] = fits ? n_items : 0;
    p.header[kHdrPrefillStages] = fits ? running : 0;
    p.header[kHdrTotalKeys] = (int)(s_decode_keys > 0x7fffffffull ? 0x7fffffffull : s_decode_keys);
  }
  if (flags && p.status) atomicOr(reinterpret_cast<unsigned*>(p.status), flags);
}

}  // namespace

cudaError_t launch_q8_plan(const Params& p, int n_sm, cudaStream_t stream, bool pdl) {
  return launch_kernel(q8_plan_kernel, dim3(1), dim3(kThreads), 0, stream, pdl, p, n_sm);
}

}  // namespace ejk
