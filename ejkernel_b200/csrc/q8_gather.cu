// Ragged attention over the 8-bit cache, the simple form: one CTA per (query token, query head), everything in float32.
//
//   x_j = scale * k_scale[j] * sum_d q[d] k[j, d];  y_j = cap * tanh(x_j / cap);  masked keys are left out
//   out[d] = sum_j exp(y_j - m) v_scale[j] v[j, d] / (sum_j exp(y_j - m) + sum_i exp(sink_i - m)),   m = max
//
// One pass over the keys in tiles of 128 with a running maximum and sum: a thread computes one key's logit, then the
// threads share out head_dim for P.V.  It asks nothing of the page size and serves what the pipelined kernels do not.
#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr int kThreads = 128;
constexpr float kLog2eG = 1.4426950408889634f;

__device__ __forceinline__ float block_reduce(float v, bool want_max, float* s_red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = want_max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();  // s_red of an earlier reduction has been read
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = want_max ? fmaxf(v, s_red[w]) : v + s_red[w];
  return v;
}

template <typename T, typename Code, int D>
__global__ void __launch_bounds__(kThreads) q8_gather_kernel(const Params p, const Q8Cache c) {
  constexpr int kCols = (D + kThreads - 1) / kThreads;  // columns of the output per thread
  __shared__ float s_q[D];
  __shared__ float s_p[kThreads];      // exp(y - m) * v_scale of the tile's keys
  __shared__ long long s_row[kThreads];  // offset of the key's V row, -1: no key
  __shared__ float s_red[kThreads / 32];
  const int t = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x;
  const int h = hq / p.G;
  T* out = reinterpret_cast<T*>(p.out) + ((size_t)t * p.Hq + hq) * D;
  unsigned flags = 0;

  int S = p.num_seqs[0];
  if (S > p.S_max) {
    S = p.S_max;
    flags |= EJK_RPA_ST_NUM_SEQS;
  }
  // the last sequence that starts at or before t: sequences without rows share their successor's start
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.query_start_loc[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int q0 = S > 0 ? p.query_start_loc[lo] : 0, q1 = S > 0 ? p.query_start_loc[lo + 1] : 0;
  if (S > 0 && bad_rows(q0, q1, p.T)) flags |= EJK_RPA_ST_QLEN;
  if (S <= 0 || t < q0 || t >= q1 || bad_rows(q0, q1, p.T)) {  // a row of no sequence, or of one whose offsets are refused
    for (int d = tid; d < D; d += kThreads) out[d] = Mma<T>::from_float(0.f);
    if (flags && tid == 0 && p.status) atomicOr(reinterpret_cast<unsigned*>(p.status), flags);
    return;
  }
  int kv_len = p.context_lens[lo];
  const int kv_cap = p.pages_per_seq * p.page_size;
  if (kv_len < 0 || kv_len > kv_cap) {
    flags |= EJK_RPA_ST_KVLEN;
    kv_len = kv_len < 0 ? 0 : kv_cap;
  }
  if (q1 - q0 > kv_len) flags |= EJK_RPA_ST_QLEN;
  const int pos = kv_len - (q1 - q0) + (t - q0);
  const int key0 = (p.window > 0 && pos - p.window + 1 > 0) ? pos - p.window + 1 : 0;
  const int key1 = pos + 1 < kv_len ? pos + 1 : kv_len;

  const T* q = reinterpret_cast<const T*>(p.q) + ((size_t)t * p.Hq + hq) * D;
  for (int d = tid; d < D; d += kThreads) s_q[d] = to_float(q[d]);
  __syncthreads();

  const int32_t* tab = p.block_tables + (size_t)lo * p.pages_per_seq;
  const int bpp = p.page_size >> c.block_shift;
  float m = -INFINITY, l = 0.f, acc[kCols] = {};
  for (int base = key0; base < key1; base += kThreads) {
    const int key = base + tid;
    float y = -INFINITY, vs = 0.f;
    long long v_row = -1;
    if (key < key1) {
      const int pi = key / p.page_size, off = key - pi * p.page_size;
      int page = tab[pi];
      if ((unsigned)page >= (unsigned)p.num_pages) {
        flags |= EJK_RPA_ST_PAGE_ID;
        page = 0;
      }
      const long long plane = ((long long)page * p.Hkv + h) * 2;
      const uint8_t* k = c.pages + (plane * p.page_size + off) * D;
      const float ks = c.scales[plane * bpp + (off >> c.block_shift)];
      vs = c.scales[(plane + 1) * bpp + (off >> c.block_shift)];
      v_row = ((plane + 1) * p.page_size + off) * D;
      float dot = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; d += 16) {
        const uint4 w = *reinterpret_cast<const uint4*>(k + d);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) dot = fmaf(Code::decode((uint8_t)(ww[i >> 2] >> (8 * (i & 3)))), s_q[d + i], dot);
      }
      dot *= ks;
      y = p.cap != 0.f ? soft_cap_large(p.cap_log2, dot * p.inv_cap_scale) : dot * p.scale_log2;
    }
    const float m_new = fmaxf(m, block_reduce(y, true, s_red));
    const float mu = m_new == -INFINITY ? 0.f : m_new;
    const float f = fast_exp2(m - mu);  // 0 on the first tile
    const float e = fast_exp2(y - mu);
    l = l * f + block_reduce(e, false, s_red);
    m = m_new;
    s_p[tid] = key < key1 ? e * vs : 0.f;
    s_row[tid] = v_row;
    __syncthreads();
    const int n = key1 - base < kThreads ? key1 - base : kThreads;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const int d = tid + i * kThreads;
      if (d >= D) continue;
      float a = acc[i] * f;
      for (int j = 0; j < n; ++j) a = fmaf(s_p[j], Code::decode(c.pages[s_row[j] + d]), a);
      acc[i] = a;
    }
    __syncthreads();
  }
  float scl = 1.f;
  if (p.num_sinks > 0) {
    // sinks join the denominator only
    const int srow = (p.sink_rows == p.Hq) ? hq : (p.sink_rows == p.Hkv ? h : 0);
    const float* sk = p.sinks + (size_t)srow * p.num_sinks;
    float sm = m;
    for (int i = 0; i < p.num_sinks; ++i) sm = fmaxf(sm, sk[i] * kLog2eG);
    const float mf = sm == -INFINITY ? 0.f : sm;
    scl = fast_exp2(m - mf);
    l *= scl;
    for (int i = 0; i < p.num_sinks; ++i) l += fast_exp2(sk[i] * kLog2eG - mf);
  }
  scl = l > 0.f ? scl / l : 0.f;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    const int d = tid + i * kThreads;
    if (d < D) out[d] = Mma<T>::from_float(acc[i] * scl);
  }
  if (flags && p.status) atomicOr(reinterpret_cast<unsigned*>(p.status), flags);
}

template <typename T, typename Code>
cudaError_t dispatch(const Params& p, const Q8Cache& c, cudaStream_t stream) {
  const dim3 grid(p.T, p.Hq);
  switch (p.D) {
    case 64: q8_gather_kernel<T, Code, 64><<<grid, kThreads, 0, stream>>>(p, c); break;
    case 128: q8_gather_kernel<T, Code, 128><<<grid, kThreads, 0, stream>>>(p, c); break;
    case 256: q8_gather_kernel<T, Code, 256><<<grid, kThreads, 0, stream>>>(p, c); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_q8_gather(const Params& p, const Q8Cache& c, int dtype, int code, cudaStream_t stream) {
  if (code == EJK_Q8_I8)
    return dtype == EJK_RPA_BF16 ? dispatch<__nv_bfloat16, CodeI8>(p, c, stream) : dispatch<__half, CodeI8>(p, c, stream);
  return dtype == EJK_RPA_BF16 ? dispatch<__nv_bfloat16, CodeE4M3>(p, c, stream) : dispatch<__half, CodeE4M3>(p, c, stream);
}

}  // namespace ejk
