// C ABI of the operators around the 8-bit cache (declared in include/ejk_q8.h).
#include <cmath>
#include <cstring>

#include "q8_types.cuh"

namespace ejk {
namespace {

__device__ int32_t g_status;  // zero when the library is loaded, one on each device

int log2_exact(int x) {
  if (x <= 0 || (x & (x - 1))) return -1;
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

// what every operator on the cache needs
int check_cache(const ejk_q8_shape& s) {
  if (s.num_pages <= 0 || s.page_size <= 0 || s.num_kv_heads <= 0) return EJK_RPA_E_SHAPE;
  if ((long long)s.num_pages * s.page_size > 0x7fffffffLL || s.num_kv_heads > 0x7fff) return EJK_RPA_E_SHAPE;
  if (s.head_dim != 64 && s.head_dim != 128 && s.head_dim != 256) return EJK_RPA_E_HEAD_DIM;
  if (s.dtype != EJK_RPA_BF16 && s.dtype != EJK_RPA_F16) return EJK_RPA_E_DTYPE;
  if (s.code_dtype != EJK_RPA_E4M3 && s.code_dtype != EJK_Q8_I8) return EJK_RPA_E_DTYPE;
  if (log2_exact(s.scale_block) < 0 || s.page_size % s.scale_block) return EJK_RPA_E_SHAPE;
  return 0;
}

Q8Cache cache_of(const void* pages, const float* scales, const ejk_q8_shape& s) {
  Q8Cache c;
  c.pages = static_cast<uint8_t*>(const_cast<void*>(pages));
  c.scales = const_cast<float*>(scales);
  c.num_pages = s.num_pages;
  c.page_size = s.page_size;
  c.Hkv = s.num_kv_heads;
  c.D = s.head_dim;
  c.block_shift = log2_exact(s.scale_block);
  return c;
}

// the checks of arguments see the call as one of ejk_rpa_launch over a 16-bit pool
ejk_rpa_shape as_rpa(const ejk_q8_shape& s) {
  return {s.total_tokens, s.max_num_seqs, s.pages_per_seq, s.num_pages, s.page_size,
          s.num_q_heads, s.num_kv_heads, s.head_dim, s.dtype, 0};
}

int check_attention(const ejk_q8_shape& s) {
  if (int e = check_cache(s)) return e;
  if (s.num_q_heads > 0xffff) return EJK_RPA_E_SHAPE;  // a grid dimension
  return check_rpa_shape(as_rpa(s));
}

// The workspace: the split-KV kernel's arrival counters, which are zero between calls, and its parts; where the batch can hold
// tensor tiles, their work list and the parts of items that are cut along KV (two tiles of 128 rows, two parts per CTA).
struct Q8Workspace {
  size_t part_ml_off, part_o_off, header_off, items_off, prefix_off, item_tickets_off, item_ml_off, item_o_off, total;
  int max_items;
};
Q8Workspace q8_workspace(const ejk_q8_shape& s, int n_sm, bool with_tiles) {
  const int G = s.num_q_heads / s.num_kv_heads;
  const size_t rt = G > 8 ? 16 : 8, slots = 2 * 2 * (size_t)n_sm;
  Q8Workspace w;
  size_t off = EJK_Q8_TICKET_BYTES;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) / 256 * 256;
    return at;
  };
  w.part_ml_off = take(slots * rt * sizeof(float2));
  w.part_o_off = take(slots * rt * s.head_dim * sizeof(float));
  if (with_tiles) {
    w.max_items = (int)((long long)s.total_tokens * G / kPrefillRows + s.max_num_seqs);
    const size_t rows = 2 * (size_t)n_sm * 2 * kPrefillRows;
    w.header_off = take(kHdrWords * sizeof(int32_t));
    w.items_off = take((size_t)w.max_items * sizeof(Unit));
    w.prefix_off = take(((size_t)w.max_items + 1) * sizeof(int32_t));
    w.item_tickets_off = take((size_t)w.max_items * s.num_kv_heads * 2 * 4 * sizeof(int32_t));
    w.item_ml_off = take(rows * sizeof(float2));
    w.item_o_off = take(rows * s.head_dim * sizeof(float));
  }
  w.total = off;
  return w;
}
// Are the tensor tiles considered?  Where the caller says from how many query tokens on they pay (num_queries_per_block), always.
// Without that only where the batch has more tokens than the tables have rows: in a table with idle rows nothing that the host
// knows tells a chunk of a prompt from a decode batch, whose calls would all pay for a plan and a tile kernel that find nothing to
// do: 128 decode requests of 1000 keys 72 -> 90 us, 4 of 100 18 -> 33 (a 2000-token prompt in a table of 4096 rows: 1085 us without
// the hint, 102 with it).
bool tiles_possible(const ejk_q8_shape& s, int num_queries_per_block) {
  return q8_prefill_supported(s.head_dim) && (num_queries_per_block > 0 || s.total_tokens > s.max_num_seqs);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
template <typename... P>
bool aligned4(P... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) == 0; }
bool finite(float x) { return x == x && !std::isinf(x); }

}  // namespace
}  // namespace ejk

using namespace ejk;

extern "C" {

size_t ejk_q8_workspace_bytes(const ejk_q8_shape* shape) { return ejk_q8_attention_workspace_bytes(shape, nullptr); }

size_t ejk_q8_attention_workspace_bytes(const ejk_q8_shape* shape, const ejk_rpa_attrs* attrs) {
  if (!shape || check_attention(*shape) != 0) return 0;
  const int n_sm = sm100_sm_count();
  if (!n_sm) return 0;
  if (kQ8TicketsPerCta * 2 * n_sm * sizeof(int32_t) > EJK_Q8_TICKET_BYTES) return 0;
  return q8_workspace(*shape, n_sm, tiles_possible(*shape, attrs ? attrs->num_queries_per_block : 0)).total;
}

int ejk_q8_status_word(int32_t** word) {
  if (!word) return EJK_RPA_E_NULL;
  *word = nullptr;
  if (!sm100_sm_count()) return EJK_RPA_E_DEVICE;
  // loading the library's image, should this be its first use, is refused to a thread that is capturing in the strict mode
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  if (cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode); e != cudaSuccess) return static_cast<int>(e);
  void* at = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&at, g_status);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return static_cast<int>(e);
  *word = static_cast<int32_t*>(at);
  return 0;
}

int ejk_q8_attention_launch(const void* queries, const void* kv_pages, const float* kv_scales,
                            const int32_t* context_lens, const int32_t* block_tables, const int32_t* query_start_loc,
                            const int32_t* num_seqs, const float* softmax_aux, void* out, void* workspace,
                            size_t workspace_bytes, int32_t* status, const ejk_q8_shape* shape,
                            const ejk_rpa_attrs* attrs, void* stream) {
  set_last_launches(0);
  if (!queries || !kv_pages || !kv_scales || !context_lens || !block_tables || !query_start_loc || !num_seqs || !out ||
      !workspace || !shape || !attrs)
    return EJK_RPA_E_NULL;
  if (int e = check_attention(*shape)) return e;
  const ejk_q8_shape& s = *shape;
  const ejk_rpa_attrs& a = *attrs;
  // with what the kernels multiply by: the scale and the cap in units of log2, and the scale in units of the cap
  const float log2e = 1.4426950408889634f;
  const float in_caps = a.logits_soft_cap != 0.f ? a.softmax_scale / a.logits_soft_cap : 0.f;
  if (!finite(a.softmax_scale * log2e) || !finite(a.logits_soft_cap) || !finite(in_caps * (2.f * log2e))) return EJK_RPA_E_ARG;
  if (std::fabs(a.logits_soft_cap) > 0x1p100f) return EJK_RPA_E_ARG;
  if (a.q_scale != 0.f || a.out_scale != 0.f) return EJK_RPA_E_ARG;
  if (a.num_sinks < 0 || (a.num_sinks > 0 && !softmax_aux)) return EJK_RPA_E_ARG;
  if (a.num_sinks > 0 && a.sink_rows != s.num_q_heads && a.sink_rows != s.num_kv_heads && a.sink_rows != 1) return EJK_RPA_E_ARG;
  if (!aligned16(queries) || !aligned16(kv_pages) || !aligned16(out)) return EJK_RPA_E_ALIGN;
  if (!aligned4(kv_scales, context_lens, block_tables, query_start_loc, num_seqs, softmax_aux, status)) return EJK_RPA_E_ALIGN;
  const int n_sm = sm100_sm_count();
  if (!n_sm) return EJK_RPA_E_DEVICE;
  if (kQ8TicketsPerCta * 2 * n_sm * sizeof(int32_t) > EJK_Q8_TICKET_BYTES) return EJK_RPA_E_DEVICE;
  const bool tiles = tiles_possible(s, a.num_queries_per_block);
  const Q8Workspace W = q8_workspace(s, n_sm, tiles);
  if (workspace_bytes < W.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return EJK_RPA_E_WORKSPACE;

  const LaunchOptions opt = launch_options();
  const bool use_tma = opt.path != 1 && q8_tma_supported(s.page_size) && std::fabs(a.logits_soft_cap) <= kPlainCap;
  if (opt.path == 2 && !use_tma) return EJK_RPA_E_ARG;

  Params p;
  std::memset(&p, 0, sizeof(p));
  p.q = queries;
  p.kv = kv_pages;
  p.context_lens = context_lens;
  p.block_tables = block_tables;
  p.query_start_loc = query_start_loc;
  p.num_seqs = num_seqs;
  p.sinks = softmax_aux;
  p.out = out;
  p.status = status;
  p.T = s.total_tokens;
  p.S_max = s.max_num_seqs;
  p.pages_per_seq = s.pages_per_seq;
  p.num_pages = s.num_pages;
  p.page_size = s.page_size;
  p.Hq = s.num_q_heads;
  p.Hkv = s.num_kv_heads;
  p.G = s.num_q_heads / s.num_kv_heads;
  p.D = p.Dq = p.Dkv = s.head_dim;
  p.window = a.sliding_window > 0 ? a.sliding_window : 0;
  p.num_sinks = a.num_sinks;
  p.sink_rows = a.sink_rows;
  p.out_scale = 1.f;
  p.scale = a.softmax_scale;
  p.scale_log2 = a.softmax_scale * log2e;
  p.cap = a.logits_soft_cap;
  p.cap_log2 = a.logits_soft_cap * log2e;
  p.inv_cap_scale = in_caps;
  const Q8Cache c = cache_of(kv_pages, kv_scales, s);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!use_tma) {
    cudaError_t e = launch_q8_gather(p, c, s.dtype, s.code_dtype, st);
    if (e != cudaSuccess) return static_cast<int>(e);
    set_last_launches(1);
    return 0;
  }

  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.tickets = reinterpret_cast<int32_t*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + W.part_ml_off);
  p.part_o = reinterpret_cast<float*>(ws + W.part_o_off);
  p.rows_per_tile = p.G > 8 ? 16 : 8;
  p.min_chunk = opt.min_chunk;
  if (a.num_kv_pages_per_block > 0) {  // per-call hint: the smallest KV chunk, in pages
    long long chunk = (long long)a.num_kv_pages_per_block * s.page_size;
    chunk = (chunk + kTileTokens - 1) / kTileTokens * kTileTokens;
    p.min_chunk = chunk > 0x40000000ll ? 0x40000000 : (int)chunk;
  }
  p.page_shift = log2_exact(s.page_size);
  // tokens per TMA box: the largest power of two that divides the page size, at most the 64 tokens that chunks are cut at
  p.tma_block_tokens = 8;
  while (p.tma_block_tokens < kTileTokens && s.page_size % (p.tma_block_tokens * 2) == 0) p.tma_block_tokens *= 2;
  p.tma_block_shift = log2_exact(p.tma_block_tokens);
  p.wait_timeout_ms = opt.wait_ms;
  p.test_withhold = opt.test_withhold;
  // Batches that can hold a sequence with many query rows also get the tensor-tile kernel; whether one qualifies is decided by the
  // planner on the device.  From 32 rows on (8 tokens at 4 heads per kv head): 64 requests of 6 tokens over 2000 keys take 160 us in
  // row tiles and 229 in tensor tiles, of 8 tokens 205 and 217, of 16 tokens 373 and 217; 8 requests over 8000 keys 92 and 125,
  // 109 and 125, 190 and 133; 128 over 500 keys 121 and 154, 139 and 137, 266 and 139.  Few short requests would gain from a higher
  // threshold (8 of 8 tokens over 2000 keys 45 and 70): num_queries_per_block is theirs.
  int prefill_rows = opt.prefill_rows;
  if (a.num_queries_per_block > 0) {  // per-call hint: query tokens from which on a sequence is served by tensor tiles
    const long long r = (long long)a.num_queries_per_block * p.G;
    prefill_rows = r > 0x40000000ll ? 0x40000000 : (int)r;
  }
  const bool use_prefill = tiles && prefill_rows > 0 && (long long)s.total_tokens * p.G >= prefill_rows;
  p.prefill_min_rows = use_prefill ? prefill_rows : 0;
  p.prefill_share = opt.prefill_share;
  if (use_prefill) {
    p.header = reinterpret_cast<int32_t*>(ws + W.header_off);
    p.punits = reinterpret_cast<Unit*>(ws + W.items_off);
    p.max_punits = W.max_items;
    p.prefill_item_rows = 2 * kPrefillRows;
    if (opt.prefill_split) {
      p.pprefix = reinterpret_cast<int32_t*>(ws + W.prefix_off);
      p.ptickets = reinterpret_cast<int32_t*>(ws + W.item_tickets_off);
      p.ppart_ml = reinterpret_cast<float2*>(ws + W.item_ml_off);
      p.ppart_o = reinterpret_cast<float*>(ws + W.item_o_off);
      p.prefill_split = opt.prefill_split;
    }
  }
  // Kernels of one call are launched as programmatic dependents: each waits on the device for what it needs of the one
  // before, the planner for whatever precedes the call.
  const bool pdl = opt.overlap != 0;
  p.pdl = pdl ? (use_prefill ? 1 : 2) : 0;
  int launches = 0;
  cudaError_t e;
  if (use_prefill) {
    e = launch_q8_plan(p, n_sm, st, pdl);
    if (e != cudaSuccess) return static_cast<int>(e);
    e = launch_q8_prefill(p, c, s.dtype, s.code_dtype, n_sm, st, pdl);
    if (e != cudaSuccess) return static_cast<int>(e);
    launches += 2;
  }
  e = launch_q8_splitkv(p, c, s.dtype, s.code_dtype, n_sm, st, pdl);
  if (e != cudaSuccess) return static_cast<int>(e);
  ++launches;
  set_last_launches(launches);
  return 0;
}

int ejk_q8_write_launch(const void* keys, const void* values, int64_t key_stride, int64_t value_stride, void* kv_pages,
                        float* kv_scales, const int32_t* slots, int32_t* status, const ejk_q8_shape* shape, void* stream) {
  set_last_launches(0);
  if (!keys || !values || !kv_pages || !kv_scales || !slots || !shape) return EJK_RPA_E_NULL;
  if (int e = check_cache(*shape)) return e;
  const ejk_q8_shape& s = *shape;
  if (s.total_tokens <= 0) return EJK_RPA_E_SHAPE;
  const int64_t row = (int64_t)s.num_kv_heads * s.head_dim;
  if (key_stride < row || value_stride < row) return EJK_RPA_E_SHAPE;
  if (!aligned16(keys) || !aligned16(values) || !aligned16(kv_pages) || key_stride % 8 || value_stride % 8) return EJK_RPA_E_ALIGN;
  if (!aligned4(kv_scales, slots, status)) return EJK_RPA_E_ALIGN;
  if (!sm100_sm_count()) return EJK_RPA_E_DEVICE;
  cudaError_t e = launch_q8_write(keys, values, key_stride, value_stride, cache_of(kv_pages, kv_scales, s), slots, status,
                                  s.total_tokens, s.dtype, s.code_dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return static_cast<int>(e);
  set_last_launches(1);
  return 0;
}

int ejk_q8_read_launch(const void* kv_pages, const float* kv_scales, const int32_t* slots, void* keys, void* values,
                       int32_t* status, const ejk_q8_shape* shape, void* stream) {
  set_last_launches(0);
  if (!keys || !values || !kv_pages || !kv_scales || !slots || !shape) return EJK_RPA_E_NULL;
  if (int e = check_cache(*shape)) return e;
  const ejk_q8_shape& s = *shape;
  // the kernel counts 8-element chunks of K in 32 bits
  if (s.total_tokens <= 0 || (long long)s.total_tokens * s.num_kv_heads * (s.head_dim / 8) > 0x7fffffffLL) return EJK_RPA_E_SHAPE;
  if (!aligned16(keys) || !aligned16(values) || !aligned16(kv_pages) || !aligned4(kv_scales, slots, status)) return EJK_RPA_E_ALIGN;
  if (!sm100_sm_count()) return EJK_RPA_E_DEVICE;
  cudaError_t e = launch_q8_read(cache_of(kv_pages, kv_scales, s), slots, keys, values, status, s.total_tokens, s.dtype,
                                 s.code_dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return static_cast<int>(e);
  set_last_launches(1);
  return 0;
}

int ejk_page_tables_launch(const int32_t* query_lens, const int32_t* context_lens, int32_t* block_tables,
                           int32_t* free_pages, const int32_t* num_free, const int32_t* num_seqs, const uint8_t* finished,
                           int32_t* new_context_lens, int32_t* query_start_loc, int32_t* slots, int32_t* new_num_free,
                           int32_t* status, int32_t max_num_seqs, int32_t pages_per_seq, int32_t page_size,
                           int32_t capacity, int32_t total_tokens, void* stream) {
  set_last_launches(0);
  if (!query_lens || !context_lens || !block_tables || !free_pages || !num_free || !num_seqs || !new_context_lens ||
      !query_start_loc || !new_num_free || (total_tokens > 0 && !slots))
    return EJK_RPA_E_NULL;
  if (max_num_seqs <= 0 || max_num_seqs > kPageTableMaxRows || pages_per_seq <= 0 || page_size <= 0 || capacity <= 0 || total_tokens < 0)
    return EJK_RPA_E_SHAPE;
  if ((long long)pages_per_seq * page_size > 0x3fffffffLL || total_tokens > 0x3fffffff) return EJK_RPA_E_SHAPE;
  if (!aligned4(query_lens, context_lens, block_tables, free_pages, num_free, num_seqs, new_context_lens, query_start_loc, slots, new_num_free, status))
    return EJK_RPA_E_ALIGN;
  if (!sm100_sm_count()) return EJK_RPA_E_DEVICE;
  cudaError_t e = launch_page_tables(query_lens, context_lens, block_tables, free_pages, num_free, num_seqs, finished,
                                     new_context_lens, query_start_loc, slots, new_num_free, status, max_num_seqs,
                                     pages_per_seq, page_size, capacity, total_tokens, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return static_cast<int>(e);
  set_last_launches(1);
  return 0;
}

}  // extern "C"
