// Page tables and slot maps of one serving step from the requests' lengths (the definition is in ejk_q8.h).
//
// With c = context length, q = new tokens, g = page size:
//   held = ceil(c / g), need = ceil((c + q) / g) - held, and exclusive sums over the rows: start (of q), first (of need),
//   back (of held, finished rows only).  The stack holds n' = num_free + sum(back) pages after the returns;
//   table[row, held + j] = stack[n' - 1 - (first + j)] where first + need <= n'.
// The sums are one block's scans, 1024 rows at a time; the pages of a round are then written one thread per page (a
// binary search over the round's sums finds the row), so that one long prompt does not serialise on one thread.
#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr int kRows = 1024;
constexpr int kSlotThreads = 256;

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

// exclusive sum of v over the block, and its total
__device__ long long block_scan(long long v, long long* s_warp, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s_warp of an earlier scan has been read
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long y = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    s_warp[lane] = y;
  }
  __syncthreads();
  total = s_warp[31];
  return x - v + (warp ? s_warp[warp - 1] : 0);
}

struct Row {
  int c, q, held, need;
  bool gone, ok;  // ok: lengths within the contract and the row's table
};

__device__ __forceinline__ Row load_row(const TableArgs& a, int s, int S, unsigned& flags) {
  Row r = {0, 0, 0, 0, false, true};
  if (s >= S) return r;
  r.c = a.context_lens[s];
  r.gone = a.finished && a.finished[s] != 0;
  r.q = r.gone ? 0 : a.query_lens[s];
  const long long cap = (long long)a.pps * a.page;
  if (r.c < 0 || r.c > cap) {
    flags |= EJK_RPA_ST_KVLEN;
    r.ok = r.gone;  // a finished row gives back what its table holds
    r.c = r.c < 0 ? 0 : (int)cap;
  }
  if (r.q < 0) {
    flags |= EJK_RPA_ST_QLEN;
    r.q = 0;
  }
  r.held = (r.c + a.page - 1) / a.page;
  if ((long long)r.c + r.q > cap) {
    flags |= EJK_RPA_ST_KVLEN;
    r.ok = false;
  }
  if (r.ok && !r.gone) r.need = (int)(((long long)r.c + r.q + a.page - 1) / a.page) - r.held;
  return r;
}

__global__ void __launch_bounds__(kRows) page_tables_kernel(const TableArgs a) {
  __shared__ long long s_warp[32];
  __shared__ long long s_ex[kRows];
  __shared__ int s_held[kRows];
  __shared__ unsigned char s_ok[kRows];
  __shared__ unsigned long long s_taken;
  const int tid = threadIdx.x;
  unsigned flags = 0;
  int S = a.num_seqs[0];
  if (S > a.S) {
    S = a.S;
    flags |= EJK_RPA_ST_NUM_SEQS;
  }
  if (S < 0) S = 0;
  long long n = a.num_free[0];
  if (n < 0 || n > a.capacity) {
    flags |= EJK_Q8_ST_POOL;
    n = n < 0 ? 0 : a.capacity;
  }
  if (tid == 0) s_taken = 0;
  // the row of page j of a round: the last row whose sum is not above j (rows without pages share their successor's)
  auto find = [&](long long j, int rows) {
    int lo = 0, hi = rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_ex[mid] <= j) lo = mid;
      else hi = mid;
    }
    return lo;
  };

  // ---- returned pages go on top
  if (a.finished) {
    for (int s0 = 0; s0 < S; s0 += kRows) {
      unsigned f = 0;
      const Row r = load_row(a, s0 + tid, S, f);
      long long total;
      s_ex[tid] = block_scan(r.gone ? r.held : 0, s_warp, total);
      __syncthreads();
      const int rows = S - s0 < kRows ? S - s0 : kRows;
      for (long long j = tid; j < total; j += kRows) {
        const int i = find(j, rows);
        const long long at = n + j;
        if (at < a.capacity) a.free_pages[at] = a.tables[(size_t)(s0 + i) * a.pps + (j - s_ex[i])];
        else flags |= EJK_Q8_ST_POOL;
      }
      n += total;
      __syncthreads();  // s_ex; and the pages are visible to the threads that take them below
    }
    if (n > a.capacity) n = a.capacity;
  }

  // ---- starts, lengths, new pages
  long long start = 0, first = 0;
  for (int s0 = 0; s0 < S; s0 += kRows) {
    const int s = s0 + tid;
    Row r = load_row(a, s, S, flags);
    long long q_total, need_total;
    const long long q0 = start + block_scan(r.q, s_warp, q_total);
    const long long p0 = block_scan(r.need, s_warp, need_total);
    if (q0 + r.q > a.T) {  // the batch is longer than its buffers
      flags |= EJK_RPA_ST_QLEN;
      r.ok = false;
    }
    if (first + p0 + r.need > n) {
      if (r.need > 0) flags |= EJK_Q8_ST_POOL;
      r.ok = r.ok && r.need == 0;
    }
    const bool takes = r.ok && !r.gone;
    if (s < S) {
      a.starts[s] = (int)(q0 < a.T ? q0 : a.T);
      a.new_lens[s] = r.gone ? 0 : (takes ? r.c + r.q : r.c);
    }
    if (takes && r.need > 0) atomicAdd(&s_taken, (unsigned long long)r.need);
    s_ex[tid] = p0;
    s_held[tid] = r.held;
    s_ok[tid] = takes;
    __syncthreads();
    const int rows = S - s0 < kRows ? S - s0 : kRows;
    for (long long j = tid; j < need_total; j += kRows) {
      const int i = find(j, rows);
      const long long at = n - 1 - (first + j);
      if (s_ok[i] && at >= 0) a.tables[(size_t)(s0 + i) * a.pps + s_held[i] + (j - s_ex[i])] = a.free_pages[at];
    }
    start += q_total;
    first += need_total;
    __syncthreads();
  }
  for (int s = S + tid; s < a.S; s += kRows) a.new_lens[s] = 0;
  for (int s = S + tid; s <= a.S; s += kRows) a.starts[s] = (int)(start < a.T ? start : a.T);
  if (tid == 0) a.new_free[0] = (int)(n - (long long)s_taken);
  if (flags && a.status) atomicOr(reinterpret_cast<unsigned*>(a.status), flags);
}

// slots[t] of every token from the finished tables: one thread per token, a binary search for its row
__global__ void __launch_bounds__(kSlotThreads) slot_map_kernel(const TableArgs a) {
  const int t = blockIdx.x * kSlotThreads + threadIdx.x;
  if (t >= a.T) return;
  int S = a.num_seqs[0];
  S = S > a.S ? a.S : S;
  int slot = -1;
  unsigned flags = 0;
  if (S > 0 && t < a.starts[S]) {
    int lo = 0, hi = S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int c = a.context_lens[lo], q = a.query_lens[lo];
    if (c >= 0 && q > 0 && a.new_lens[lo] == c + q) {  // the row was served
      const int pos = c + t - a.starts[lo];
      const int pi = pos / a.page;
      if (pos >= 0 && pos < c + q && pi < a.pps) {
        const long long at = (long long)a.tables[(size_t)lo * a.pps + pi] * a.page + (pos - pi * a.page);
        if (at >= 0 && at <= 0x7fffffffLL) slot = (int)at;
        else flags |= EJK_RPA_ST_PAGE_ID;
      }
    }
  }
  a.slots[t] = slot;
  if (flags && a.status) atomicOr(reinterpret_cast<unsigned*>(a.status), flags);
}

}  // namespace

cudaError_t launch_page_tables(const int32_t* query_lens, const int32_t* context_lens, int32_t* tables, int32_t* free_pages,
                               const int32_t* num_free, const int32_t* num_seqs, const uint8_t* finished,
                               int32_t* new_lens, int32_t* starts, int32_t* slots, int32_t* new_free, int32_t* status,
                               int S, int pps, int page, int capacity, int T, cudaStream_t st) {
  const TableArgs a = {query_lens, context_lens, tables, free_pages, num_free, num_seqs, finished, new_lens, starts,
                       slots, new_free, status, S, pps, page, capacity, T};
  page_tables_kernel<<<1, kRows, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || T == 0) return e;
  slot_map_kernel<<<(T + kSlotThreads - 1) / kSlotThreads, kSlotThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace ejk
