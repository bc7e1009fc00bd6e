// Page tables and slot maps of one serving step from the requests' lengths (the definition is in ejk_q8.h).
//
// With c = context length, q = new tokens, g = page size, per row:
//   held = ceil(c / g), need = ceil((c + q) / g) - held, and exclusive sums over the rows: start (of q), first (of need),
//   back (of held, finished rows only).  The stack holds n' = num_free + sum(back) pages after the returns;
//   page i of the new ones is stack[n' - 1 - i], and row s takes the pages first .. first + need - 1 where they exist.
//
// A few bytes per token and page: launches and latency bound it, so it is one kernel.  Every block computes the three sums
// of all rows in its own shared memory (a few microseconds that they all spend at the same time, instead of a second
// launch behind the first) and then writes its share of the tokens, the new pages and the returned ones.  That needs no order
// between blocks, because nothing is read that this call writes: a new page that comes from a finished row is looked up
// in that row's table, not on the stack, and the slots of new pages are computed, not read back.
// Measured on the device: 4 rows 4.2 us, 1000 rows with 9 thousand tokens and 25 thousand returned pages 9.6 us (one block for the
// sums and pages and a second kernel for the slots: 6.9 and 37.6 us).
#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr unsigned kMaxSum = 0x7fffffffu;  // sums saturate here: above every token, page and stack count there is

struct TableArgs {
  const int32_t* query_lens;
  const int32_t* context_lens;
  int32_t* tables;
  int32_t* free_pages;
  const int32_t* num_free;
  const int32_t* num_seqs;
  const uint8_t* finished;  // may be null
  int32_t* new_lens;
  int32_t* starts;
  int32_t* slots;
  int32_t* new_free;
  int32_t* status;  // may be null
  int32_t S, pps, page, capacity, T;
};

__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, kMaxSum); }  // associative for a, b <= kMaxSum

struct Row {
  int c, q, held, need;
  bool gone, ok;  // ok: lengths within the contract and the row's table
};

__device__ __forceinline__ Row load_row(const TableArgs& a, int s, unsigned& flags) {
  Row r;
  r.c = a.context_lens[s];
  r.q = a.query_lens[s];
  r.gone = a.finished && a.finished[s] != 0;
  r.ok = true;
  r.need = 0;
  if (r.gone) r.q = 0;
  const int cap = a.pps * a.page;  // below 2^30
  if (r.c < 0 || r.c > cap) {
    flags |= EJK_RPA_ST_KVLEN;
    r.ok = false;
    r.c = r.c < 0 ? 0 : cap;
  }
  if (r.q < 0) {
    flags |= EJK_RPA_ST_QLEN;
    r.q = 0;
  }
  r.held = (r.c + a.page - 1) / a.page;
  if (r.q > cap - r.c) {
    flags |= EJK_RPA_ST_KVLEN;
    r.ok = false;
  }
  if (r.ok && !r.gone) r.need = (r.c + r.q + a.page - 1) / a.page - r.held;
  return r;
}

// exclusive sums of three counters over the block's threads, and the totals
__device__ void block_scan(unsigned (&v)[3], unsigned (&total)[3], unsigned (*s_warp)[3]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
  unsigned inc[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    unsigned x = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = sat_add(x, y);
    }
    inc[k] = x;
    if (lane == 31) s_warp[warp][k] = x;
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      unsigned x = lane < n_warps ? s_warp[lane][k] : 0u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = sat_add(x, y);
      }
      if (lane < n_warps) s_warp[lane][k] = x;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    unsigned before = __shfl_up_sync(0xffffffffu, inc[k], 1);
    if (lane == 0) before = 0u;
    v[k] = sat_add(before, warp ? s_warp[warp - 1][k] : 0u);
    total[k] = s_warp[n_warps - 1][k];
  }
}

__global__ void __launch_bounds__(1024) page_tables_kernel(const TableArgs a) {
  extern __shared__ unsigned s_sums[];  // start[S] first[S] back[S]
  __shared__ unsigned s_warp[32][3];
  __shared__ unsigned s_taken;
  const int tid = threadIdx.x, n_threads = blockDim.x;
  unsigned flags = 0;
  int S = a.num_seqs[0];
  if (S > a.S) {
    S = a.S;
    flags |= EJK_RPA_ST_NUM_SEQS;
  }
  if (S < 0) S = 0;
  unsigned* start = s_sums;
  unsigned* first = s_sums + S;
  unsigned* back = s_sums + 2 * S;
  int n_free = a.num_free[0];
  if (n_free < 0 || n_free > a.capacity) {
    flags |= EJK_Q8_ST_POOL;
    n_free = n_free < 0 ? 0 : a.capacity;
  }
  if (tid == 0) s_taken = 0;

  // ---- the sums: neighbouring rows to a thread, then across threads
  const int per = (S + n_threads - 1) / n_threads;
  const int s0 = min(tid * per, S), s1 = min(s0 + per, S);
  unsigned v[3] = {0u, 0u, 0u}, total[3];
  for (int s = s0; s < s1; ++s) {
    const Row r = load_row(a, s, flags);
    v[0] = sat_add(v[0], (unsigned)r.q);
    v[1] = sat_add(v[1], (unsigned)r.need);
    v[2] = sat_add(v[2], r.gone ? (unsigned)r.held : 0u);
  }
  block_scan(v, total, s_warp);
  const unsigned returned = total[2];
  unsigned n_all = sat_add((unsigned)n_free, returned);  // pages on the stack once the returned ones are on it
  if (n_all > (unsigned)a.capacity) {
    flags |= EJK_Q8_ST_POOL;
    n_all = (unsigned)a.capacity;
  }
  // is a row with these sums served?
  auto served = [&](const Row& r, unsigned q0, unsigned p0, unsigned& f) {
    if (r.gone) return false;
    bool ok = r.ok;
    if (sat_add(q0, (unsigned)r.q) > (unsigned)a.T) {  // the batch is longer than its buffers
      f |= EJK_RPA_ST_QLEN;
      ok = false;
    }
    if (r.need > 0 && sat_add(p0, (unsigned)r.need) > n_all) {
      f |= EJK_Q8_ST_POOL;
      ok = false;
    }
    return ok;
  };
  for (int s = s0; s < s1; ++s) {
    unsigned none = 0;
    const Row r = load_row(a, s, none);
    start[s] = v[0];
    first[s] = v[1];
    back[s] = v[2];
    const bool ok = served(r, v[0], v[1], flags);
    if (blockIdx.x == 0) {
      a.starts[s] = (int)min(v[0], (unsigned)a.T);
      a.new_lens[s] = r.gone ? 0 : (ok ? r.c + r.q : r.c);
      if (ok && r.need > 0) atomicAdd(&s_taken, (unsigned)r.need);
    }
    v[0] = sat_add(v[0], (unsigned)r.q);
    v[1] = sat_add(v[1], (unsigned)r.need);
    v[2] = sat_add(v[2], r.gone ? (unsigned)r.held : 0u);
  }
  __syncthreads();
  const unsigned q_total = min(total[0], (unsigned)a.T);
  if (blockIdx.x == 0) {
    for (int s = S + tid; s < a.S; s += n_threads) a.new_lens[s] = 0;
    for (int s = S + tid; s <= a.S; s += n_threads) a.starts[s] = (int)q_total;
    if (tid == 0) a.new_free[0] = (int)(n_all - s_taken);
  }

  // the last row whose sum is not above j: rows without a share have their successor's sum
  auto find = [&](const unsigned* sum, unsigned j) {
    int lo = 0, hi = S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sum[mid] <= j) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  // page `j` of the returned ones, and page `i` from the top of the stack
  auto returned_page = [&](unsigned j) {
    const int s = find(back, j);
    return a.tables[(size_t)s * a.pps + (j - back[s])];
  };
  auto top_page = [&](unsigned i) {
    const unsigned at = n_all - 1u - i;
    return at < (unsigned)n_free ? a.free_pages[at] : returned_page(at - (unsigned)n_free);
  };
  const unsigned gid = blockIdx.x * n_threads + tid, n_grid = gridDim.x * n_threads;

  // ---- slots
  for (unsigned t = gid; t < (unsigned)a.T; t += n_grid) {
    int slot = -1;
    if (t < q_total) {
      const int s = find(start, t);
      unsigned none = 0;
      const Row r = load_row(a, s, none);
      if (served(r, start[s], first[s], none)) {
        const int pos = r.c + (int)(t - start[s]);
        const int pi = pos / a.page;
        const int page = pi < r.held ? a.tables[(size_t)s * a.pps + pi] : top_page(first[s] + (unsigned)(pi - r.held));
        const long long at = (long long)page * a.page + (pos - pi * a.page);
        if (at >= 0 && at <= 0x7fffffffLL) slot = (int)at;
        else flags |= EJK_RPA_ST_PAGE_ID;
      }
    }
    a.slots[t] = slot;
  }
  // ---- new pages into the tables
  for (unsigned j = gid; j < min(total[1], n_all); j += n_grid) {
    const int s = find(first, j);
    unsigned none = 0;
    const Row r = load_row(a, s, none);
    if (served(r, start[s], first[s], none)) a.tables[(size_t)s * a.pps + r.held + (j - first[s])] = top_page(j);
  }
  // ---- returned pages onto the stack
  for (unsigned j = gid; j < n_all - min(n_all, (unsigned)n_free); j += n_grid) a.free_pages[(unsigned)n_free + j] = returned_page(j);
  if (flags && a.status) atomicOr(reinterpret_cast<unsigned*>(a.status), flags);
}

}  // namespace

cudaError_t launch_page_tables(const int32_t* query_lens, const int32_t* context_lens, int32_t* tables, int32_t* free_pages,
                               const int32_t* num_free, const int32_t* num_seqs, const uint8_t* finished,
                               int32_t* new_lens, int32_t* starts, int32_t* slots, int32_t* new_free, int32_t* status,
                               int S, int pps, int page, int capacity, int T, cudaStream_t st) {
  const TableArgs a = {query_lens, context_lens, tables, free_pages, num_free, num_seqs, finished, new_lens, starts,
                       slots, new_free, status, S, pps, page, capacity, T};
  const size_t smem = (size_t)S * 3 * sizeof(unsigned);
  if (smem > 32 * 1024) {
    // The limit of the kernel on the current device, set whenever it may be needed: two words of host work.  Without it a block
    // gets 48 KB, of which the kernel's own few hundred bytes take a part
    if (cudaError_t e = cudaFuncSetAttribute(page_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPageTableMaxRows * 12); e != cudaSuccess)
      return e;
  }
  // a small block synchronises faster; as many blocks as leave each thread a handful of tokens and pages
  const int threads = S <= 256 ? 256 : 1024;
  const long long work = (long long)T + 8ll * S;
  long long blocks = (work + threads - 1) / threads;
  if (blocks > 128) blocks = 128;
  page_tables_kernel<<<(int)blocks, threads, smem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace ejk
