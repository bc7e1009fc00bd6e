// Write and read of the 8-bit cache (the definitions are in ejk_q8.h).
#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr int kWriteThreads = 128;
constexpr int kReadThreads = 256;

template <int N>
struct Vec16;  // N 16-bit elements
template <>
struct Vec16<2> { using type = uint32_t; };
template <>
struct Vec16<4> { using type = uint2; };
template <>
struct Vec16<8> { using type = uint4; };
template <int N>
struct Vec8;  // N bytes
template <>
struct Vec8<2> { using type = uint16_t; };
template <>
struct Vec8<4> { using type = uint32_t; };
template <>
struct Vec8<8> { using type = uint2; };

// One CTA per row of the batch; a row that does not open a scale block of the batch has nothing to do.  A warp takes
// one (head, K or V) of the block at a time: it sweeps the block's new rows twice (they are in L1 the second time),
// for the largest value and for the codes.
template <typename T, typename Code, int D>
__global__ void __launch_bounds__(kWriteThreads)
q8_write_kernel(const T* __restrict__ keys, const T* __restrict__ values, long long key_stride, long long value_stride,
                const Q8Cache c, const int32_t* __restrict__ slots, int32_t* status, int n_rows) {
  constexpr int E = D / 32;  // elements per lane
  using V16 = typename Vec16<E>::type;
  using V8 = typename Vec8<E>::type;
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slot = slots[t];
  if (slot < 0) return;
  const int n_slots = c.num_pages * c.page_size;
  unsigned flags = 0;
  if (slot >= n_slots) {
    if (threadIdx.x == 0 && status) atomicOr(reinterpret_cast<unsigned*>(status), EJK_RPA_ST_PAGE_ID);
    return;
  }
  const int block = slot >> c.block_shift;
  if (t > 0) {
    const int before = slots[t - 1];
    if (before >= 0 && before < n_slots && (before >> c.block_shift) == block) return;
  }
  // rows t .. t + n - 1 share the block
  int n = 1;
  while (true) {
    const int i = t + n + lane;
    const int s = i < n_rows ? slots[i] : -1;
    const unsigned same = __ballot_sync(0xffffffffu, s >= 0 && s < n_slots && (s >> c.block_shift) == block);
    const int run = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
    n += run;
    if (run < 32) break;
  }
  const int first = slot & ((1 << c.block_shift) - 1);  // rows [0, first) of the block are kept
  const int page = slot / c.page_size;
  const int bpp = c.page_size >> c.block_shift;
  const int sub = (slot - page * c.page_size) >> c.block_shift;
  const int off0 = sub << c.block_shift;  // offset of the block inside its page

  for (int hk = warp; hk < 2 * c.Hkv; hk += kWriteThreads / 32) {
    const int h = hk >> 1, kv = hk & 1;
    const long long stride = kv ? value_stride : key_stride;
    const T* src = (kv ? values : keys) + (long long)t * stride + h * D + lane * E;
    const long long plane = ((long long)page * c.Hkv + h) * 2 + kv;
    uint8_t* dst = c.pages + (plane * c.page_size + off0) * D + lane * E;
    float* scale_at = c.scales + plane * bpp + sub;

    float amax = 0.f;
    bool odd = false;
    for (int r = 0; r < n; ++r) {
      const V16 w = *reinterpret_cast<const V16*>(src + r * stride);
      const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float a = fabsf(to_float(x[i]));
        if (a <= 3.4028234663852886e38f) amax = fmaxf(amax, a);
        else odd = true;  // NaN or infinity
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (odd) flags |= EJK_Q8_ST_NONFINITE;
    float scale = power_of_two_scale<Code>(amax);
    if (first > 0) {
      const float old = *scale_at;
      if (old >= scale) {
        scale = old;
      } else {
        // the kept rows move to the larger scale; the quotient of the scales is a power of two, or a rounded one
        // where the old scale was not
        const float ratio = old / scale;
        for (int r = 0; r < first; ++r) {
          V8* at = reinterpret_cast<V8*>(dst + (long long)r * D);
          V8 w = *at;
          uint8_t* b = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
          for (int i = 0; i < E; ++i) b[i] = Code::encode(Code::decode(b[i]) * ratio);
          *at = w;
        }
      }
    }
    __syncwarp();
    if (lane == 0) *scale_at = scale;
    // a scale that this kernel wrote is a power of two, and the product with its inverse is the quotient; one that a
    // caller put there need not be
    const bool exact = (__float_as_uint(scale) & 0x7fffffu) == 0;
    const float inv = exact ? power_of_two_inverse(scale) : 0.f;
    for (int r = 0; r < n; ++r) {
      const V16 w = *reinterpret_cast<const V16*>(src + r * stride);
      const T* x = reinterpret_cast<const T*>(&w);
      V8 o;
      uint8_t* b = reinterpret_cast<uint8_t*>(&o);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float v = to_float(x[i]);
        v = exact ? v * inv : v / scale;
        v = v == v ? fminf(fmaxf(v, -Code::kMax), Code::kMax) : 0.f;
        b[i] = Code::encode(v);
      }
      const int off = slots[t + r] & ((1 << c.block_shift) - 1);
      *reinterpret_cast<V8*>(dst + (long long)off * D) = o;
    }
  }
  if (flags && status) atomicOr(reinterpret_cast<unsigned*>(status), flags);
}

// Eight elements of a row per thread.
template <typename T, typename Code>
__global__ void __launch_bounds__(kReadThreads)
q8_read_kernel(const Q8Cache c, const int32_t* __restrict__ slots, uint4* __restrict__ keys, uint4* __restrict__ values,
               int32_t* status, long long n_chunks, int chunks_per_row) {
  constexpr float kBig = sizeof(T) == 2 && std::is_same<T, __half>::value ? 65504.f : 3.3895313892515355e38f;
  const long long i = (long long)blockIdx.x * kReadThreads + threadIdx.x;
  if (i >= n_chunks) return;
  const long long row = i / chunks_per_row;  // (token, head, K or V)
  const int ch = (int)(i - row * chunks_per_row);
  const int kv = (int)(row & 1);
  const long long th = row >> 1;
  const long long t = th / c.Hkv;
  const int h = (int)(th - t * c.Hkv);
  const int slot = slots[t];
  uint4 o = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= c.num_pages * c.page_size) {
    if (status) atomicOr(reinterpret_cast<unsigned*>(status), EJK_RPA_ST_PAGE_ID);
  } else if (slot >= 0) {
    const int page = slot / c.page_size, off = slot - page * c.page_size;
    const long long plane = ((long long)page * c.Hkv + h) * 2 + kv;
    const uint2 w = *reinterpret_cast<const uint2*>(c.pages + (plane * c.page_size + off) * c.D + ch * 8);
    const float s = c.scales[plane * (c.page_size >> c.block_shift) + (off >> c.block_shift)];
    const uint8_t* b = reinterpret_cast<const uint8_t*>(&w);
    uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x0 = fminf(fmaxf(Code::decode(b[2 * j]) * s, -kBig), kBig);
      const float x1 = fminf(fmaxf(Code::decode(b[2 * j + 1]) * s, -kBig), kBig);
      ow[j] = Mma<T>::pack(x0, x1);
    }
  }
  (kv ? values : keys)[th * chunks_per_row + ch] = o;
}

template <typename T, typename Code>
cudaError_t write_dispatch(const void* keys, const void* values, long long ks, long long vs, const Q8Cache& c,
                           const int32_t* slots, int32_t* status, int rows, cudaStream_t st) {
  const T* k = static_cast<const T*>(keys);
  const T* v = static_cast<const T*>(values);
  switch (c.D) {
    case 64: q8_write_kernel<T, Code, 64><<<rows, kWriteThreads, 0, st>>>(k, v, ks, vs, c, slots, status, rows); break;
    case 128: q8_write_kernel<T, Code, 128><<<rows, kWriteThreads, 0, st>>>(k, v, ks, vs, c, slots, status, rows); break;
    case 256: q8_write_kernel<T, Code, 256><<<rows, kWriteThreads, 0, st>>>(k, v, ks, vs, c, slots, status, rows); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

template <typename T, typename Code>
cudaError_t read_dispatch(const Q8Cache& c, const int32_t* slots, void* keys, void* values, int32_t* status, int rows,
                          cudaStream_t st) {
  const int cpr = c.D / 8;
  const long long n = (long long)rows * c.Hkv * 2 * cpr;
  q8_read_kernel<T, Code><<<(unsigned)((n + kReadThreads - 1) / kReadThreads), kReadThreads, 0, st>>>(
      c, slots, static_cast<uint4*>(keys), static_cast<uint4*>(values), status, n, cpr);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_q8_write(const void* keys, const void* values, long long key_stride, long long value_stride,
                            const Q8Cache& c, const int32_t* slots, int32_t* status, int rows, int dtype, int code,
                            cudaStream_t st) {
  if (code == EJK_Q8_I8)
    return dtype == EJK_RPA_BF16 ? write_dispatch<__nv_bfloat16, CodeI8>(keys, values, key_stride, value_stride, c, slots, status, rows, st)
                                 : write_dispatch<__half, CodeI8>(keys, values, key_stride, value_stride, c, slots, status, rows, st);
  return dtype == EJK_RPA_BF16 ? write_dispatch<__nv_bfloat16, CodeE4M3>(keys, values, key_stride, value_stride, c, slots, status, rows, st)
                               : write_dispatch<__half, CodeE4M3>(keys, values, key_stride, value_stride, c, slots, status, rows, st);
}

cudaError_t launch_q8_read(const Q8Cache& c, const int32_t* slots, void* keys, void* values, int32_t* status, int rows,
                           int dtype, int code, cudaStream_t st) {
  if (code == EJK_Q8_I8)
    return dtype == EJK_RPA_BF16 ? read_dispatch<__nv_bfloat16, CodeI8>(c, slots, keys, values, status, rows, st)
                                 : read_dispatch<__half, CodeI8>(c, slots, keys, values, status, rows, st);
  return dtype == EJK_RPA_BF16 ? read_dispatch<__nv_bfloat16, CodeE4M3>(c, slots, keys, values, status, rows, st)
                               : read_dispatch<__half, CodeE4M3>(c, slots, keys, values, status, rows, st);
}

}  // namespace ejk
