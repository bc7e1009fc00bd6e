// Write and read of the 8-bit cache (the definitions are in ejk_q8.h).
#include <type_traits>

#include "q8_types.cuh"

namespace ejk {
namespace {

constexpr int kWriteThreads = 128;
constexpr int kReadThreads = 256;

// Codes of eight floats.  The fast form takes finite values within the codes' range; the careful one clamps and writes NaN as 0.
template <typename Code, bool CAREFUL>
__device__ __forceinline__ uint2 encode8(const float (&x)[8]) {
  uint32_t two[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
    if (CAREFUL) {
      a = a == a ? fminf(fmaxf(a, -Code::kMax), Code::kMax) : 0.f;
      b = b == b ? fminf(fmaxf(b, -Code::kMax), Code::kMax) : 0.f;
    }
    two[i] = Code::encode2(a, b);
  }
  return make_uint2(prmt(two[0], two[1], 0x5410u), prmt(two[2], two[3], 0x5410u));
}
template <typename T>
__device__ __forceinline__ float2 floats_of(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// One (head, K or V) of one scale block, by one warp: rows t .. t + n - 1 of the batch.  A lane holds eight elements, so that a
// warp takes 4, 2 or 1 rows at a time (head_dim 64, 128, 256).  At most ROWS of them are read once, into registers, for the
// largest value and for the codes; of a larger block the rest is read twice, the second time from L2.
template <typename T, typename Code, int D, int ROWS, typename Offset>
__device__ __forceinline__ unsigned write_block(const T* __restrict__ src, long long stride, uint8_t* dst, float* scale_at,
                                                int first, int n, Offset offset) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;         // lanes per row, rows at a time
  constexpr int IT = (ROWS + RPI - 1) / RPI;
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x & 31, lr = lane / LPR, ch = lane % LPR;
  src += (long long)lr * stride + ch * 8;
  dst += ch * 8;
  unsigned flags = 0;
  const float old = first > 0 ? *scale_at : 0.f;
  auto row = [&](int r0) { return *reinterpret_cast<const uint4*>(src + (long long)r0 * stride); };
  uint4 w[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) w[i] = i * RPI + lr < n ? row(i * RPI) : make_uint4(0u, 0u, 0u, 0u);
  // the largest |x|, as 16-bit patterns: finite values order like integers
  uint32_t top = 0;
  auto larger = [&](const uint4& v) {
    top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
  };
#pragma unroll
  for (int i = 0; i < IT; ++i) larger(w[i]);
  for (int r = IT * RPI; r + lr < n; r += RPI) larger(row(r));
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  const bool odd = top >= kInf;  // a NaN or an infinity among them: the largest of the others, element by element
  if (odd) {
    flags |= EJK_Q8_ST_NONFINITE;
    top = 0;
    for (int r = 0; r + lr < n; r += RPI) {
      const uint4 v = row(r);
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = x[i] & 0x7fffu, hi = (x[i] >> 16) & 0x7fffu;
        if (lo < kInf) top = max(top, lo);
        if (hi < kInf) top = max(top, hi);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  const unsigned short top16 = (unsigned short)top;
  float scale = power_of_two_scale<Code>(to_float(*reinterpret_cast<const T*>(&top16)));
  if (first > 0) {
    if (old >= scale) {
      scale = old;
    } else {
      // the kept rows move to the larger scale; the quotient of the scales is a power of two, or a rounded one
      // where the old scale was not
      const float ratio = old / scale;
      for (int r0 = 0; r0 < first; r0 += 8 * RPI) {
        uint2 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + i * RPI + lr;
          if (r < first) v[i] = *reinterpret_cast<const uint2*>(dst + (long long)r * D);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = r0 + i * RPI + lr;
          if (r < first) {
            uint32_t h[4];
            Code::widen(v[i].x, h[0], h[1]);
            Code::widen(v[i].y, h[2], h[3]);
            float x[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
              x[2 * k] = f.x * ratio;
              x[2 * k + 1] = f.y * ratio;
            }
            *reinterpret_cast<uint2*>(dst + (long long)r * D) = encode8<Code, false>(x);
          }
        }
      }
    }
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale_at = scale;
  // a scale that this kernel wrote is a power of two up to 2^122, and the product with its inverse is the quotient; one that a
  // caller put there need not be, or be 2^127, whose inverse is no normal number
  const bool exact = (__float_as_uint(scale) & 0x7fffffu) == 0 && __float_as_uint(scale) < (254u << 23);
  const float inv = exact ? power_of_two_inverse(scale) : 0.f;
  auto put = [&](const uint4& v, int r) {
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
    float f[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 two = floats_of<T>(x[k]);
      f[2 * k] = two.x;
      f[2 * k + 1] = two.y;
    }
    uint2 o;
    if (exact && !odd) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= inv;
      o = encode8<Code, false>(f);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = f[k] / scale;
      o = encode8<Code, true>(f);
    }
    *reinterpret_cast<uint2*>(dst + (long long)offset(r) * D) = o;
  };
#pragma unroll
  for (int i = 0; i < IT; ++i)
    if (i * RPI + lr < n) put(w[i], i * RPI + lr);
  for (int r = IT * RPI + lr; r < n; r += RPI) put(row(r - lr), r);
  return flags;
}

// A block of the batch is found by its first row: row t opens one if row t - 1 is elsewhere.  A CTA looks through `window` rows
// for such rows -- one in short batches, where every row may open a block and parallelism is what counts, more in long ones,
// where most rows open none and most CTAs would start for nothing -- and a warp of it takes one (head, K or V).
// DRAM bounds the long batches (2 bytes in, 1 byte out per element), the chain slots -> rows -> codes the short ones:
// 11629 f16 rows of 8 heads of 128 to int8 in blocks of 32 (71 MB) 17.5 us = 4.1 TB/s, 256 decode tokens 5.2 us, one token 1.9 us.
template <typename T, typename Code, int D>
__global__ void __launch_bounds__(kWriteThreads)
q8_write_kernel(const T* __restrict__ keys, const T* __restrict__ values, long long key_stride, long long value_stride,
                const Q8Cache c, const int32_t* __restrict__ slots, int32_t* status, int n_rows, int window) {
  constexpr int ROWS = D == 256 ? 16 : 32;  // rows held in registers
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hk = blockIdx.y * (kWriteThreads / 32) + warp;
  if (hk >= 2 * c.Hkv) return;
  const int h = hk >> 1, kv = hk & 1;
  const int n_slots = c.num_pages * c.page_size;
  const int block_mask = (1 << c.block_shift) - 1;
  const int bpp = c.page_size >> c.block_shift;
  unsigned flags = 0;
  // scale block of a slot; -1: the row is skipped, or out of range
  auto block_of = [&](int s) { return s >= 0 && s < n_slots ? s >> c.block_shift : -1; };
  const int t0 = blockIdx.x * window;
  // lane i looks at row t0 + i
  const int slot_l = t0 + lane < n_rows ? slots[t0 + lane] : -1;
  const int slot_b = lane == 0 && t0 > 0 ? slots[t0 - 1] : -1;
  const int mine = block_of(slot_l);
  int before = __shfl_up_sync(0xffffffffu, mine, 1);
  if (lane == 0) before = block_of(slot_b);
  if (lane < window && slot_l >= n_slots) flags |= EJK_RPA_ST_PAGE_ID;
  unsigned openers = __ballot_sync(0xffffffffu, lane < window && mine >= 0 && mine != before);

  while (openers) {
    const int at = __ffs(openers) - 1, t = t0 + at;
    openers &= openers - 1;
    const int slot = __shfl_sync(0xffffffffu, slot_l, at), block = slot >> c.block_shift;
    // rows t .. t + n - 1 share the block
    const unsigned other = __ballot_sync(0xffffffffu, mine != block) >> at;
    int n = other ? __ffs(other) - 1 : 32 - at;
    if (at + n == 32) {
      while (true) {
        const int i = t + n + lane;
        const unsigned same = __ballot_sync(0xffffffffu, block_of(i < n_rows ? slots[i] : -1) == block);
        const int run = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
        n += run;
        if (run < 32) break;
      }
    }
    const int first = slot & block_mask;  // rows [0, first) of the block are kept
    const int page = slot / c.page_size;
    const int sub = (slot - page * c.page_size) >> c.block_shift;
    const long long stride = kv ? value_stride : key_stride;
    const T* src = (kv ? values : keys) + (long long)t * stride + h * D;
    const long long plane = ((long long)page * c.Hkv + h) * 2 + kv;
    uint8_t* dst = c.pages + (plane * c.page_size + (sub << c.block_shift)) * D;
    float* scale_at = c.scales + plane * bpp + sub;
    // Offsets of the rows in the block: slots ascend, so that they are neighbours if the last one is n - 1 further
    int last = __shfl_sync(0xffffffffu, slot_l, (at + n - 1) & 31);
    if (at + n > 32) last = slots[t + n - 1];
    const bool dense = last - slot == n - 1;
    auto offset = [&](int r) { return dense ? first + r : slots[t + r] & block_mask; };
    if (n == 1) flags |= write_block<T, Code, D, 1>(src, stride, dst, scale_at, first, n, offset);
    else flags |= write_block<T, Code, D, ROWS>(src, stride, dst, scale_at, first, n, offset);
  }
  if (flags && status) atomicOr(reinterpret_cast<unsigned*>(status), flags);
}

__device__ __forceinline__ float clamp_keep_nan(float x, float big) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(x), "f"(big));
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(r), "f"(-big));
  return r;
}

// Eight elements of K and of V of two rows per thread: four independent 8-byte loads in flight, 16-byte stores.  DRAM bounds
// it: 65536 rows of 8 heads of 128 (403 MB) 75.8 us = 5.3 TB/s, 0.82 of the measured copy rate (one 8-byte load per
// thread: 136 us).
template <typename T, typename Code>
__global__ void __launch_bounds__(kReadThreads)
q8_read_kernel(const Q8Cache c, const int32_t* __restrict__ slots, uint4* __restrict__ keys, uint4* __restrict__ values,
               int32_t* status, int n_rows, int chunk_shift) {
  constexpr float kBig = std::is_same<T, __half>::value ? 65504.f : 3.3895313892515355e38f;
  const unsigned per_row = (unsigned)c.Hkv << chunk_shift;  // 8-element chunks of K in a row
  const unsigned half_rows = ((unsigned)n_rows + 1) / 2;
  const unsigned i = blockIdx.x * kReadThreads + threadIdx.x;
  const unsigned row = i / per_row;
  if (row >= half_rows) return;
  const unsigned u = i - row * per_row, h = u >> chunk_shift, ch = u & ((1u << chunk_shift) - 1u);
  const int n_slots = c.num_pages * c.page_size;
  const int bpp = c.page_size >> c.block_shift;
  uint2 code[2][2];
  float scale[2][2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const unsigned t = row + j * half_rows;
    const int slot = t < (unsigned)n_rows ? slots[t] : -1;
    if (slot >= n_slots && status) atomicOr(reinterpret_cast<unsigned*>(status), EJK_RPA_ST_PAGE_ID);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      code[j][kv] = make_uint2(0u, 0u);
      scale[j][kv] = 0.f;
    }
    if (slot >= 0 && slot < n_slots) {
      const int page = slot / c.page_size, off = slot - page * c.page_size;
      const long long plane = ((long long)page * c.Hkv + h) * 2;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        code[j][kv] = __ldg(reinterpret_cast<const uint2*>(c.pages + ((plane + kv) * c.page_size + off) * c.D + ch * 8));
        scale[j][kv] = __ldg(c.scales + (plane + kv) * bpp + (off >> c.block_shift));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const unsigned t = row + j * half_rows;
    if (t >= (unsigned)n_rows) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint4 o;
      uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
      const uint32_t w[2] = {code[j][kv].x, code[j][kv].y};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t lo, hi;
        Code::widen(w[k], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        const float s = scale[j][kv];
        ow[2 * k] = Mma<T>::pack(clamp_keep_nan(a.x * s, kBig), clamp_keep_nan(a.y * s, kBig));
        ow[2 * k + 1] = Mma<T>::pack(clamp_keep_nan(b.x * s, kBig), clamp_keep_nan(b.y * s, kBig));
      }
      (kv ? values : keys)[(size_t)t * per_row + u] = o;
    }
  }
}

template <typename T, typename Code>
cudaError_t write_dispatch(const void* keys, const void* values, long long ks, long long vs, const Q8Cache& c,
                           const int32_t* slots, int32_t* status, int rows, cudaStream_t st) {
  const T* k = static_cast<const T*>(keys);
  const T* v = static_cast<const T*>(values);
  // rows that a CTA looks through: up to 1024 rows one each, then what keeps about as many windows (12 thousand rows in blocks of
  // 32: 24 us with windows of 32, 20 us with 16)
  int window = 1;
  while (window < 32 && window < (1 << c.block_shift) && rows / window > 1024) window *= 2;
  const dim3 grid((rows + window - 1) / window, (2 * c.Hkv + kWriteThreads / 32 - 1) / (kWriteThreads / 32));
  switch (c.D) {
    case 64: q8_write_kernel<T, Code, 64><<<grid, kWriteThreads, 0, st>>>(k, v, ks, vs, c, slots, status, rows, window); break;
    case 128: q8_write_kernel<T, Code, 128><<<grid, kWriteThreads, 0, st>>>(k, v, ks, vs, c, slots, status, rows, window); break;
    case 256: q8_write_kernel<T, Code, 256><<<grid, kWriteThreads, 0, st>>>(k, v, ks, vs, c, slots, status, rows, window); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

template <typename T, typename Code>
cudaError_t read_dispatch(const Q8Cache& c, const int32_t* slots, void* keys, void* values, int32_t* status, int rows,
                          cudaStream_t st) {
  int chunk_shift = 3;  // log2 of the 8-element chunks of head_dim 64, 128, 256
  while ((8 << chunk_shift) < c.D) ++chunk_shift;
  const long long n = (long long)((rows + 1) / 2) * c.Hkv << chunk_shift;
  q8_read_kernel<T, Code><<<(unsigned)((n + kReadThreads - 1) / kReadThreads), kReadThreads, 0, st>>>(
      c, slots, static_cast<uint4*>(keys), static_cast<uint4*>(values), status, rows, chunk_shift);
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
